"""What is measured of the operators an attention rank runs around the routed experts: the block-scaled FP8 linear,
the FP8 shared expert, the router and the balance loss.

``run`` with ``own`` false computes each in plain torch operations; with ``own`` true it makes the calls a user
makes (``asap_b200.linear.Fp8Linear`` / ``Fp8SharedExpert``, ``asap_b200.router.route`` / ``balance_loss``).
Sizes: hidden 7168 / intermediate 2048 / 256 experts top-8 sigmoid and hidden 8192 / intermediate 3584 / 64 experts
top-6 softmax are the layers the benchmark serves; hidden 1024 / intermediate 512 / 16 experts top-2 is the small one.

Activations are quantised per row and block of 128 values along K, scale = amax / 448 with amax at least 1e-10.
Weight scales in fp32: codes = e4m3(x * (448 / amax)), the quotient and the product each rounded to fp32 as part of
the format.  Weight scales in E8M0: the activation scale is rounded up to a power of two and codes = e4m3(x / scale).
"""

import math
import os
import random
import sys

import torch

own = False

_MAX_MNK = 16384 * 4096 * 7168  # the largest listed linear


# ------------------------------------------------------------------------------------------------------- the cases
def _linear(m, k, n, scales, dtype):
    return {"op": "linear", "m": m, "k": k, "n": n, "scales": scales, "dtype": dtype}


def _shared(m, hidden, inter, scales, limit=0.0):
    return {"op": "shared", "m": m, "hidden": hidden, "inter": inter, "scales": scales, "limit": limit}


def _route(t, e, k, scoring, dtype, *, bias=False, groups=1, top_groups=1, renormalize=True, scale=1.0, valid=None,
           masked=0, train=False):
    return {"op": "route", "t": t, "e": e, "k": k, "scoring": scoring, "dtype": dtype, "bias": bias, "groups": groups,
            "top_groups": top_groups, "renormalize": renormalize, "scale": scale, "valid": t if valid is None else valid,
            "masked": masked, "train": train}


def _balance(t, e, k, scoring, dtype, *, sequences=1, tail=0, masked=0):
    return {"op": "balance", "t": t, "e": e, "k": k, "scoring": scoring, "dtype": dtype, "sequences": sequences,
            "tail": tail, "masked": masked}


def listed():
    return [
        # one token through the gate/up product of the shared expert: the weights' bytes are the cost
        dict(_linear(1, 7168, 4096, "fp32", "bf16"), name="linear-one-token"),
        # a decode batch of an odd size through the down product, power-of-two scales
        dict(_linear(129, 2048, 7168, "e8m0", "bf16"), name="linear-decode-batch"),
        # generic sizes that end inside a block of 128 in every dimension, fp16
        dict(_linear(1003, 2064, 1040, "fp32", "fp16"), name="linear-ragged"),
        # a prefill chunk of the hidden-8192 layer's gate/up product
        dict(_linear(8192, 8192, 7168, "fp32", "bf16"), name="linear-prefill"),
        # the largest dispatch chunk through the hidden-7168 gate/up product, power-of-two scales
        dict(_linear(16384, 7168, 4096, "e8m0", "bf16"), name="linear-prefill-pow2"),
        # the shared expert of a few decoding requests
        dict(_shared(4, 7168, 2048, "fp32"), name="shared-decode"),
        # the shared expert of the largest dispatch chunk, computed while the routed experts are away
        dict(_shared(16384, 7168, 2048, "fp32"), name="shared-prefill"),
        # the router of one decoding token: latency
        dict(_route(1, 256, 8, "sigmoid", "fp32", bias=True, groups=8, top_groups=4, scale=2.5),
             name="route-one-token"),
        # the router of a dispatch chunk padded to its bucket, group-limited with a selection bias
        dict(_route(16384, 256, 8, "sigmoid", "fp32", bias=True, groups=8, top_groups=4, scale=2.5, valid=16001),
             name="route-prefill"),
        # a training step of the 64-expert router: weights, ids and the logits' gradient
        dict(_route(8191, 64, 6, "softmax", "bf16", train=True), name="route-train"),
        # balance loss, counts and gradient over a packed batch of ragged sequences with padding behind them
        dict(_balance(16384, 256, 8, "sigmoid", "fp32", sequences=37, tail=101), name="balance-packed"),
        # the same of the small layer, one sequence
        dict(_balance(512, 16, 2, "softmax", "fp32"), name="balance-small"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "shared", "route", "route", "balance"])
    if op == "linear":
        m = _log_int(rng, 1, 16384)
        k = 16 * _log_int(rng, 16, 512) if rng.random() < 0.5 else 128 * _log_int(rng, 4, 64)
        n = 16 * _log_int(rng, 8, 512) if rng.random() < 0.5 else 128 * _log_int(rng, 2, 64)
        m = max(1, min(m, _MAX_MNK // (n * k)))
        return _linear(m, k, n, rng.choice(["fp32", "e8m0"]), rng.choice(["bf16", "bf16", "fp16"]))
    if op == "shared":
        hidden, inter = rng.choice([(1024, 512), (7168, 2048), (8192, 3584)])
        m = max(1, min(_log_int(rng, 1, 16384), 16384 * 7168 * 2048 // (hidden * inter)))
        return _shared(m, hidden, inter, rng.choice(["fp32", "e8m0"]), rng.choice([0.0, 0.0, 7.0]))
    e, k = rng.choice([(16, 2), (64, 6), (256, 8), (rng.randint(8, 512), rng.randint(1, 8))])
    t, dtype = _log_int(rng, 1, 16384), rng.choice(["fp32", "bf16"])
    scoring = rng.choice(["softmax", "sigmoid"])
    t = max(1, min(t, 16384 * 256 // e))
    masked = rng.choice([0, 0, e // 4])
    if op == "route":
        groups, top_groups = rng.choice([(1, 1), (8, 4)]) if e % 8 == 0 and e // 8 * 4 >= k else (1, 1)
        return _route(t, e, k, scoring, dtype, bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                      renormalize=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]),
                      valid=rng.choice([t, rng.randint(0, t)]), masked=masked, train=rng.random() < 0.5)
    return _balance(t, e, k, scoring, dtype, sequences=_log_int(rng, 1, max(1, t // 8)),
                    tail=rng.choice([0, t // 10]), masked=masked)


# ------------------------------------------------------------------------------------------------------ the inputs
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sgl-afd-plugin_b200")
    if root not in sys.path:
        sys.path.insert(0, root)


def _hidden(gen, m, k, dtype):
    """Normalised hidden states: unit normal with a gain per channel, a few channels an order larger."""
    gain = torch.exp(0.5 * torch.randn(k, device="cuda", generator=gen))
    gain[torch.randint(0, k, (max(1, k // 512),), device="cuda", generator=gen)] *= 10.0
    return (torch.randn(m, k, device="cuda", generator=gen) * gain).to(dtype)


def _weight(gen, n, k, scales):
    """N(0, 0.02) weights quantised per block of 128 x 128 -> (E4M3 codes [n, k], scales [n/128, k/128] rounded up)."""
    nb, kb = -(-n // 128), -(-k // 128)
    w = torch.zeros(nb * 128, kb * 128, device="cuda")
    w[:n, :k] = 0.02 * torch.randn(n, k, device="cuda", generator=gen)
    blocks = w.view(nb, 128, kb, 128)
    # blocks differ in size, as the layers' columns do
    blocks *= torch.exp2(2.0 * torch.rand(nb, 1, kb, 1, device="cuda", generator=gen) - 1.0)
    scale = blocks.abs().amax(dim=(1, 3)).clamp_min(1e-12) / 448.0
    if scales == "e8m0":
        scale = torch.exp2(torch.ceil(torch.log2(scale)))
    codes = (blocks / scale[:, None, :, None]).clamp(-448.0, 448.0).view(nb * 128, kb * 128)[:n, :k]
    if scales == "e8m0":
        scale = scale.to(torch.float8_e8m0fnu)
    return codes.to(torch.float8_e4m3fn).contiguous(), scale


def _logits(gen, t, e, dtype, masked):
    """Router logits of experts that differ in popularity; ``masked`` experts are switched off, and then one row in
    64 has no expert left."""
    logits = torch.randn(t, e, device="cuda", generator=gen) + 0.5 * torch.randn(e, device="cuda", generator=gen)
    if masked:
        logits[:, torch.randperm(e, device="cuda", generator=gen)[:masked]] = float("-inf")
        logits[torch.rand(t, device="cuda", generator=gen) < 1.0 / 64] = float("-inf")
    return logits.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    st = dict(case)
    dtype = _DTYPES[case.get("dtype", "bf16")]
    if case["op"] == "linear":
        st["x"] = _hidden(gen, case["m"], case["k"], dtype)
        st["w"], st["w_scale"] = _weight(gen, case["n"], case["k"], case["scales"])
        if own:
            _package()
            from asap_b200.linear import Fp8Linear
            st["layer"] = Fp8Linear(st["w"], st["w_scale"])
    elif case["op"] == "shared":
        st["x"] = _hidden(gen, case["m"], case["hidden"], dtype)
        st["w13"], st["w13_scale"] = _weight(gen, 2 * case["inter"], case["hidden"], case["scales"])
        st["w2"], st["w2_scale"] = _weight(gen, case["hidden"], case["inter"], case["scales"])
        if own:
            _package()
            from asap_b200.linear import Fp8SharedExpert
            st["layer"] = Fp8SharedExpert(st["w13"], st["w13_scale"], st["w2"], st["w2_scale"],
                                          swiglu_limit=case["limit"])
    elif case["op"] == "route":
        t, e, k = case["t"], case["e"], case["k"]
        st["logits"] = _logits(gen, t, e, dtype, case["masked"]).requires_grad_(case["train"])
        st["bias_t"] = 0.1 * torch.randn(e, device="cuda", generator=gen) if case["bias"] else None
        st["num_tokens"] = torch.tensor([case["valid"]], dtype=torch.int32, device="cuda") \
            if case["valid"] != t else None
        if case["train"]:
            st["grad"] = torch.randn(t, k, device="cuda", generator=gen)
    else:
        t, e, k = case["t"], case["e"], case["k"]
        logits = _logits(gen, t, e, dtype, case["masked"])
        top = torch.sort(logits.float(), dim=1, descending=True, stable=True)
        st["ids"] = torch.where(torch.isneginf(top.values[:, :k]), -1, top.indices[:, :k]).to(torch.int32).contiguous()
        st["logits"] = logits.requires_grad_(True)
        rng = random.Random(seed)
        cuts = sorted(rng.randint(0, t - case["tail"]) for _ in range(case["sequences"] - 1))
        st["cu_seqlens"] = torch.tensor([0] + cuts + [t - case["tail"]], dtype=torch.int32, device="cuda") \
            if case["sequences"] > 1 or case["tail"] else None
        st["coef"] = 1e-2
    return st


# --------------------------------------------------------------------------------------------------- the plain form
def _quantized(x, pow2):
    """[m, k] -> the values its E4M3 codes and scales stand for, fp32 [m, k]."""
    m, k = x.shape
    b = torch.zeros(m, -(-k // 128) * 128, device=x.device, dtype=torch.float32)
    b[:, :k] = x.float()
    b = b.view(m, -1, 128)
    amax = b.abs().amax(dim=2, keepdim=True).clamp_min(1e-10).double()
    if pow2:
        frac, exp = torch.frexp(amax / 448.0)
        scale = torch.ldexp(torch.ones_like(frac), exp - (frac == 0.5).to(exp.dtype)).float()
        inv = 1.0 / scale
    else:
        scale, inv = (amax / 448.0).float(), (448.0 / amax).float()
    codes = (b * inv).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return (codes.float() * scale).view(m, -1)[:, :k]


def _dequantized(w, scale):
    n, k = w.shape
    full = scale.float().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return w.float() * full


def _plain_linear(st):
    return (_quantized(st["x"], st["scales"] == "e8m0") @ _dequantized(st["w"], st["w_scale"]).t()).to(st["x"].dtype)


def _plain_shared(st):
    pow2 = st["scales"] == "e8m0"
    gu = _quantized(st["x"], pow2) @ _dequantized(st["w13"], st["w13_scale"]).t()
    g, u = gu[:, :st["inter"]], gu[:, st["inter"]:]
    if st["limit"] > 0:
        g, u = g.clamp(max=st["limit"]), u.clamp(-st["limit"], st["limit"])
    h = g / (1.0 + torch.exp(-g)) * u
    return (_quantized(h, pow2) @ _dequantized(st["w2"], st["w2_scale"]).t()).to(st["x"].dtype)


def _scores(logits, scoring):
    """(selected scores in the logits' own width, 0 where the logit is -inf)."""
    off = torch.isneginf(logits)
    if scoring == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits))
    top = logits.amax(dim=1, keepdim=True)
    ex = torch.exp(torch.where(off, torch.zeros_like(logits), logits - top)) * ~off
    return ex / ex.sum(dim=1, keepdim=True).clamp_min(1e-300 if logits.dtype == torch.float64 else 1e-38)


def _plain_route(st):
    logits, k, e = st["logits"].detach(), st["k"], st["e"]
    t = logits.shape[0]
    l64 = logits.double()  # the selection compares values that may lie close together
    s = _scores(l64, st["scoring"])
    off = torch.isneginf(l64)
    if st["num_tokens"] is not None:
        off = off | (torch.arange(t, device=off.device)[:, None] >= st["num_tokens"])
    bias = st["bias_t"]
    sel = (l64 if bias is None else s + bias.double()).masked_fill(off, float("-inf"))
    if st["groups"] > 1:
        g = torch.sort(sel.view(t, st["groups"], -1), dim=2, descending=True).values
        if bias is None:
            score = g[:, :, 0]
        else:
            score = torch.where(torch.isneginf(g[:, :, :2]), 0.0, g[:, :, :2]).sum(2)
            score = score.masked_fill(torch.isneginf(g[:, :, 0]), float("-inf"))
        kept = torch.sort(score, dim=1, descending=True, stable=True).indices[:, :st["top_groups"]]
        drop = torch.ones(t, st["groups"], dtype=torch.bool, device=sel.device).scatter_(1, kept, False)
        sel = sel.masked_fill(drop.repeat_interleave(e // st["groups"], 1), float("-inf"))
    top = torch.sort(sel, dim=1, descending=True, stable=True)
    none = torch.isneginf(top.values[:, :k])
    ids = torch.where(none, -1, top.indices[:, :k]).to(torch.int32)
    s_top = s.gather(1, top.indices[:, :k]).masked_fill(none, 0.0)
    norm = s_top.sum(1, keepdim=True) + 1e-20 if st["renormalize"] else torch.ones_like(s_top[:, :1])
    weights = (st["scale"] * s_top / norm).float()
    if not st["train"]:
        return weights, ids
    # weights -> scores -> logits; the ids carry no gradient
    grad = st["grad"].masked_fill(none, 0.0)
    s32, s_top, norm = _scores(logits.float(), st["scoring"]), s_top.float(), norm.float()
    ds_top = st["scale"] / norm * grad
    if st["renormalize"]:
        ds_top = ds_top - st["scale"] / norm * (grad * s_top).sum(1, keepdim=True) / norm
    ds = torch.zeros_like(s32).scatter_add(1, ids.clamp_min(0).long(), ds_top.masked_fill(none, 0.0))
    if st["scoring"] == "sigmoid":
        dl = s32 * (1.0 - s32) * ds
    else:
        dl = s32 * (ds - (ds * s32).sum(1, keepdim=True))
    return weights, ids, dl.to(logits.dtype)


def _plain_balance(st):
    logits, ids, e, k = st["logits"].detach(), st["ids"], st["e"], st["k"]
    t = logits.shape[0]
    cu = st["cu_seqlens"] if st["cu_seqlens"] is not None else torch.tensor([0, t], dtype=torch.int32, device="cuda")
    n_seq = cu.numel() - 1
    seq = torch.searchsorted(cu[1:].contiguous(), torch.arange(t, dtype=torch.int32, device="cuda"), right=True)
    live = (seq < n_seq) & (ids >= 0).any(1)
    seq = seq.clamp_max(n_seq - 1)
    hit = (ids >= 0) & live[:, None]
    counts = torch.zeros(n_seq * e, dtype=torch.int32, device="cuda")
    counts.scatter_add_(0, (seq[:, None] * e + ids.clamp_min(0)).reshape(-1), hit.to(torch.int32).reshape(-1))
    counts = counts.view(n_seq, e)
    tokens = torch.zeros(n_seq, device="cuda").scatter_add_(0, seq, live.float())
    p = _scores(logits.float(), st["scoring"])
    s = p
    if st["scoring"] == "sigmoid":
        s = p.masked_fill(torch.isneginf(logits), 0.0)
        p = s / s.sum(1, keepdim=True).clamp_min(1e-38)
    n = tokens.clamp_min(1.0)
    a = st["coef"] / (tokens > 0).sum().clamp_min(1) * (e / k) * counts.float() / (n * n)[:, None]
    a_row = a[seq] * live[:, None]
    dot = (a_row * p).sum(1, keepdim=True)
    loss = dot.double().sum().float()
    dl = p * (a_row - dot)
    if st["scoring"] == "sigmoid":
        dl = dl * (1.0 - s)
    return loss, counts, dl.to(logits.dtype)


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    st = state
    if not own:
        return {"linear": _plain_linear, "shared": _plain_shared, "route": _plain_route,
                "balance": _plain_balance}[st["op"]](st)
    if st["op"] in ("linear", "shared"):
        return st["layer"](st["x"])
    from asap_b200.router import balance_loss, route

    if st["op"] == "route":
        top = route(st["logits"], st["k"], scoring=st["scoring"], bias=st["bias_t"], num_groups=st["groups"],
                    top_groups=st["top_groups"], renormalize=st["renormalize"], routed_scaling_factor=st["scale"],
                    num_tokens=st["num_tokens"])
        if not st["train"]:
            return top.topk_weights, top.topk_ids
        (dl,) = torch.autograd.grad(top.topk_weights, st["logits"], st["grad"])
        return top.topk_weights.detach(), top.topk_ids, dl
    loss, counts = balance_loss(st["logits"], st["ids"], scoring=st["scoring"], coef=st["coef"],
                                cu_seqlens=st["cu_seqlens"])
    (dl,) = torch.autograd.grad(loss, st["logits"])
    return loss.detach(), counts, dl


def work(case):
    c = case
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        scale = (4 if c["scales"] == "fp32" else 1) * -(-n // 128) * -(-k // 128)
        return {"bytes": 2 * m * k + n * k + scale + 2 * m * n, "flops": 2 * m * n * k}
    if c["op"] == "shared":
        m, h, i = c["m"], c["hidden"], c["inter"]
        scale = (4 if c["scales"] == "fp32" else 1) * 3 * (h // 128) * (i // 128)
        return {"bytes": 4 * m * h + 3 * h * i + scale, "flops": 6 * m * h * i}
    t, e, k = c["t"], c["e"], c["k"]
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "route":
        back = t * k * 4 + t * e * size if c["train"] else 0
        rows = c["valid"]  # rows behind the valid ones are not read
        return {"bytes": rows * e * size + 8 * t * k + back, "flops": rows * e * (8 + k) + (4 * t * e if back else 0)}
    return {"bytes": 2 * t * e * size + 4 * t * k + 4 * c["sequences"] * (e + 1), "flops": 16 * t * e}


# ------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_codes(x, pow2, from_input):
    """Values of x's E4M3 codes, float64.  An input's quotient and product are fp32 by definition of the format; an
    intermediate is a real number."""
    m, k = x.shape
    out = torch.empty(m, k, dtype=torch.float64, device=x.device)
    for k0 in range(0, k, 128):
        b = x[:, k0:k0 + 128].double()
        amax = b.abs().max(dim=1, keepdim=True).values
        amax = torch.maximum(amax, torch.full_like(amax, torch.tensor(1e-10, dtype=torch.float32).item()))
        if pow2:
            e = torch.ceil(torch.log2(amax / 448.0))
            # log2 may round across an integer: settle by comparing
            e = torch.where(torch.exp2(e - 1) >= amax / 448.0, e - 1, e)
            e = torch.where(torch.exp2(e) < amax / 448.0, e + 1, e)
            scale = torch.exp2(e)
            q = b / scale
        elif from_input:
            scale = (amax / 448.0).float().double()
            q = (b * (448.0 / amax).float().double()).float().double()
        else:
            scale, q = amax / 448.0, b * (448.0 / amax)
        # E4M3 spacing: 2^-3 of the binade, 2^-9 below 2^-6; ties go to even
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))).clamp_min(-6.0) - 3.0)
        out[:, k0:k0 + 128] = (torch.round(q / step) * step).clamp(-448.0, 448.0) * scale
    return out


def _exact_weight(w, scale):
    s = scale.double() if scale.dtype == torch.float32 else scale.float().double()
    out = w.double()
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            out[128 * i:128 * i + 128, 128 * j:128 * j + 128] *= s[i, j]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    c, pow2 = case, case.get("scales") == "e8m0"
    if c["op"] == "linear":
        return torch.matmul(_exact_codes(st["x"], pow2, True), _exact_weight(st["w"], st["w_scale"]).T)
    if c["op"] == "shared":
        both = torch.matmul(_exact_codes(st["x"], pow2, True), _exact_weight(st["w13"], st["w13_scale"]).T)
        gate, up = both.split(c["inter"], dim=1)
        if c["limit"] > 0:
            gate, up = torch.clamp_max(gate, c["limit"]), torch.clamp(up, -c["limit"], c["limit"])
        act = gate * torch.sigmoid(gate) * up
        return torch.matmul(_exact_codes(act, pow2, False), _exact_weight(st["w2"], st["w2_scale"]).T)
    logits = st["logits"].detach().double()
    t, e, k = c["t"], c["e"], c["k"]
    dead = ~torch.isfinite(logits)
    if c["op"] == "route":
        x = logits.clone().requires_grad_(True)
        if c["scoring"] == "sigmoid":
            score = torch.sigmoid(x)
        else:
            score = torch.softmax(x.masked_fill(dead.all(1, keepdim=True), 0.0), dim=1)
        rank = logits.clone() if st["bias_t"] is None else score.detach() + st["bias_t"].double()
        closed = dead.clone()
        closed[c["valid"]:] = True
        rank[closed] = float("-inf")
        size = e // c["groups"]
        if c["groups"] > 1:
            value = []
            for g in range(c["groups"]):
                best = torch.topk(rank[:, g * size:(g + 1) * size], min(2, size), dim=1).values
                if st["bias_t"] is None:
                    value.append(best[:, 0])
                else:
                    v = torch.nan_to_num(best, neginf=0.0).sum(1)
                    value.append(torch.where(torch.isneginf(best[:, 0]), best[:, 0], v))
            order = torch.argsort(-torch.stack(value, 1), dim=1, stable=True)
            for j in range(c["top_groups"], c["groups"]):
                cols = order[:, j:j + 1] * size + torch.arange(size, device="cuda")
                rank.scatter_(1, cols, float("-inf"))
        order = torch.argsort(-rank, dim=1, stable=True)[:, :k]
        empty = torch.isneginf(rank.gather(1, order))
        picked = score.gather(1, order) * (~empty)
        w = c["scale"] * (picked / (picked.sum(1, keepdim=True) + 1e-20) if c["renormalize"] else picked)
        ids = order.masked_fill(empty, -1).to(torch.int32)
        if not c["train"]:
            return w.detach(), ids
        (dl,) = torch.autograd.grad(w, x, st["grad"].double())
        return w.detach(), ids, torch.nan_to_num(dl)
    x = logits.clone().requires_grad_(True)
    ids = st["ids"].long()
    cu = st["cu_seqlens"].tolist() if st["cu_seqlens"] is not None else [0, t]
    counts = torch.zeros(len(cu) - 1, e, dtype=torch.int32, device="cuda")
    total, filled = x.new_zeros(()), 0
    for i, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
        rows = torch.nonzero((ids[lo:hi] >= 0).any(1)).flatten() + lo
        if not rows.numel():
            continue
        filled += 1
        counts[i] = torch.bincount(ids[rows].flatten().clamp_min(-1) + 1, minlength=e + 1)[1:].to(torch.int32)
        if c["scoring"] == "softmax":
            p = torch.softmax(x[rows], dim=1)
        else:
            sig = torch.sigmoid(x[rows])
            p = sig / sig.sum(1, keepdim=True)
        total = total + (e / (k * rows.numel()) * counts[i].double() * p.mean(0)).sum()
    loss = st["coef"] * total / max(filled, 1)
    dl = torch.autograd.grad(loss, x)[0] if filled else torch.zeros_like(logits)
    return loss.detach(), counts, torch.nan_to_num(dl)
