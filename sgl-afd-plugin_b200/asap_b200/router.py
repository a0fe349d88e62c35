"""The router of an attention rank's MoE layer: which experts each token goes to and with what weights, in the form
``AsapDispatcher.dispatch`` takes, with its gradient; the balance loss over that choice; and per-expert counts.

    topk = route(logits, 8, scoring="sigmoid", bias=correction, num_groups=8, top_groups=4, routed_scaling_factor=2.5)
    out = dispatcher.combine(dispatcher.dispatch(hidden_states, topk))
    loss, counts = balance_loss(logits, topk.topk_ids, scoring="sigmoid", coef=1e-3, cu_seqlens=cu_seqlens)

The busiest F rank ends a layer's round trip, so the counts (``expert_counts``, or the loss's) say how even the F ranks'
jobs are: experts [expert_base, expert_base + num_local) are one rank's.  An F rank whose experts must not be chosen is
switched off by -inf logits (or a -inf bias) at its experts.

Logits are fp32, bf16 or fp16 [tokens, experts] with any row stride, at most 1024 experts; arithmetic is fp32, and the
selection ranks experts as unrounded scores rank (ties to the lowest expert).  Every call works on the current stream of
the logits' device and allocates what it needs from torch's caching allocator.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _native as N
from .linear import _has_tangent, _OnDevice
from .sglang_shim import StandardTopKOutput

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCORING = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS, MAX_TOPK = 1024, 32


def _check_logits(logits: torch.Tensor, scoring: str) -> None:
    if logits.dtype not in _DTYPES or logits.dim() != 2 or not logits.is_cuda:
        raise ValueError(f"logits must be a CUDA float32, bfloat16 or float16 tensor [tokens, experts], got "
                         f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid', got {scoring!r}")
    if not 1 <= logits.shape[1] <= MAX_EXPERTS:
        raise ValueError(f"need 1 to {MAX_EXPERTS} experts, got {logits.shape[1]}")
    if _has_tangent(logits):
        raise RuntimeError("the router and the balance loss have no forward-mode gradient: detach the logits")


def _rows(logits: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """Logits whose rows are contiguous, and the row stride."""
    t, e = logits.shape
    if logits.is_contiguous():
        return logits, e
    if (e > 1 and logits.stride(1) != 1) or (t > 1 and logits.stride(0) < e):
        return logits.contiguous(), e
    return logits, logits.stride(0) if t > 1 else e


def _device_int(name: str, x: torch.Tensor, like: torch.Tensor, shape) -> torch.Tensor:
    if x.dtype != torch.int32 or x.device != like.device or (shape is not None and tuple(x.shape) != tuple(shape)):
        raise ValueError(f"{name} must be int32{'' if shape is None else ' of shape ' + str(tuple(shape))} on "
                         f"{like.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.contiguous()


def _once() -> None:
    # backward runs with gradients enabled only under create_graph=True (torch's own guard costs 10 us a call)
    if torch.is_grad_enabled():
        raise RuntimeError("the router's gradients cannot be differentiated again (create_graph=True)")


def _came_back(x: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A saved tensor as backward may read it.  Its address is not the forward's: hooks unpack it elsewhere, and
    checkpointing computes it again."""
    if x.shape != shape or x.dtype is not dtype or x.device != device:
        raise RuntimeError(f"a tensor saved for the gradient came back as {x.dtype} {tuple(x.shape)} on {x.device}, was "
                           f"{dtype} {shape} on {device}")
    return x


def _route_forward(logits, opts):
    k, sigmoid, bias, groups, top_groups, renorm, scale, num_tokens = opts
    rows, ld = _rows(logits)
    t, e = rows.shape
    ids = rows.new_empty((t, k), dtype=torch.int32)
    weights = rows.new_empty((t, k), dtype=torch.float32)
    desc = N.Route_t(rows.data_ptr(), ld, _DTYPES[rows.dtype], t, e, k, sigmoid, groups, top_groups, renorm, scale, 0,
                     0 if bias is None else bias.data_ptr(), 0 if num_tokens is None else num_tokens.data_ptr())
    if t:
        with _OnDevice(rows.get_device()) as stream:
            N.run("asap_route", ctypes.byref(desc), ids.data_ptr(), weights.data_ptr(), stream)
    return weights, ids, rows, desc


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, opts):
        weights, ids, rows, desc = _route_forward(logits, opts)
        ctx.save_for_backward(rows, ids)
        # for its numbers: of its addresses, backward sets those that it reads (the bias only counts as given or not)
        ctx.desc, ctx.kind = desc, (rows.dtype, rows.device)
        ctx.mark_non_differentiable(ids)
        return weights, ids

    @staticmethod
    def backward(ctx, grad_weights, _):
        _once()
        rows, ids = ctx.saved_tensors
        desc, (dtype, device) = ctx.desc, ctx.kind
        t, e = desc.t, desc.e
        ids = _came_back(ids, (t, desc.k), torch.int32, device).contiguous()
        rows, desc.ld = _rows(_came_back(rows, (t, e), dtype, device))
        out = torch.empty_like(rows, memory_format=torch.contiguous_format)
        if t:
            desc.logits = rows.data_ptr()
            grad = grad_weights.to(torch.float32).contiguous()
            with _OnDevice(device.index) as stream:
                N.run("asap_route_backward", ctypes.byref(desc), ids.data_ptr(), grad.data_ptr(), out.data_ptr(), stream)
        return out, None


def route(logits: torch.Tensor, top_k: int, *, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
          num_groups: int = 1, top_groups: int = 1, renormalize: bool = True, routed_scaling_factor: float = 1.0,
          num_tokens: Optional[torch.Tensor] = None) -> StandardTopKOutput:
    """logits [T, E] -> StandardTopKOutput(topk_weights fp32 [T, top_k], topk_ids int32 [T, top_k], logits), best first.

    Scores are the row's softmax or its sigmoids.  Selection is by score + ``bias`` (fp32 [E], the load-balancing
    correction; it does not enter the weights), with ``num_groups`` > 1 only among the ``top_groups`` best of that many
    equal runs of experts: a group counts its best expert's score, or with a bias the sum of its two best.  weight =
    routed_scaling_factor * score, divided by the sum of the selected scores + 1e-20 if ``renormalize``.

    An expert whose logit is -inf is never chosen.  Places left over hold id -1 and weight 0, which the dispatch skips;
    so do all rows from ``num_tokens`` (int32 [1] on the device) on, the padding of a captured batch.  A row with a NaN
    logit gets NaN weights.  The weights carry a gradient to the logits (not to the bias): 0 in rows that chose no
    expert, NaN in other rows with a NaN logit."""
    _check_logits(logits, scoring)
    t, e = logits.shape
    if not 1 <= top_k <= min(e, MAX_TOPK):
        raise ValueError(f"top_k must be from 1 to {min(e, MAX_TOPK)}, got {top_k}")
    if not 1 <= num_groups <= 32 or e % num_groups or not 1 <= top_groups <= num_groups:
        raise ValueError(f"need 1 to 32 equal groups and 1 <= top_groups <= num_groups, got {top_groups} of {num_groups} "
                         f"groups of {e} experts")
    if t > 1 << 24:
        raise ValueError(f"at most {1 << 24} tokens, got {t}")
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (e,) or bias.device != logits.device:
            raise ValueError(f"bias must be float32 [{e}] on {logits.device}, got {bias.dtype} {tuple(bias.shape)} on "
                             f"{bias.device}")
        if not bias.is_contiguous():
            bias = bias.detach().contiguous()
    if num_tokens is not None:
        num_tokens = _device_int("num_tokens", num_tokens if num_tokens.dim() == 1 else num_tokens.reshape(-1), logits,
                                 (1,))
    opts = (top_k, _SCORING[scoring], bias, num_groups, top_groups, int(renormalize), float(routed_scaling_factor),
            num_tokens)
    if logits.requires_grad and torch.is_grad_enabled():
        weights, ids = _Route.apply(logits, opts)
    else:
        weights, ids = _route_forward(logits, opts)[:2]
    return StandardTopKOutput(weights, ids, logits)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, sigmoid, coef, cu_seqlens, seqs):
        rows, ld = _rows(logits)
        t, e = rows.shape
        nbytes = N.lib().asap_balance_ws_bytes(t, seqs)
        # the counts and, 8-byte aligned behind them, the workspace: one allocation, and one region to clear
        pad = seqs * e & 1
        buf = rows.new_empty(pad + seqs * e + (nbytes + 3) // 4, dtype=torch.int32)
        counts = buf.as_strided((seqs, e), (e, 1), pad)
        ctx.counts_at, ctx.ws_at = 4 * pad, 4 * (pad + seqs * e)  # bytes into buf
        ws = buf.data_ptr() + ctx.ws_at
        loss = rows.new_empty((), dtype=torch.float32)
        desc = N.Balance_t(rows.data_ptr(), ld, _DTYPES[rows.dtype], t, e, ids.shape[1], sigmoid, seqs, coef, 0,
                           ids.data_ptr(), 0 if cu_seqlens is None else cu_seqlens.data_ptr(), counts.data_ptr())
        with _OnDevice(rows.get_device()) as stream:
            N.run("asap_balance_loss", ctypes.byref(desc), ws, nbytes, loss.data_ptr(), stream)
        ctx.save_for_backward(rows, buf)  # the workspace says which tokens count, and where: ids and offsets are not needed
        # for its numbers: of its addresses, backward sets those that it reads
        ctx.desc, ctx.nbytes, ctx.kind = desc, nbytes, (buf.numel(), rows.dtype, rows.device)
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _):
        _once()
        rows, buf = ctx.saved_tensors  # (refuses what has changed since, the counts among it)
        desc, (words, dtype, device) = ctx.desc, ctx.kind
        rows, desc.ld = _rows(_came_back(rows, (desc.t, desc.e), dtype, device))
        buf = _came_back(buf, (words,), torch.int32, device).contiguous()
        if buf.data_ptr() & 7:  # the workspace in it has 8-byte words
            buf = buf.clone()
        out = torch.empty_like(rows, memory_format=torch.contiguous_format)
        desc.logits, desc.counts = rows.data_ptr(), buf.data_ptr() + ctx.counts_at
        grad = grad_loss.to(torch.float32).contiguous()
        with _OnDevice(device.index) as stream:
            N.run("asap_balance_backward", ctypes.byref(desc), buf.data_ptr() + ctx.ws_at, ctx.nbytes, grad.data_ptr(),
                  out.data_ptr(), stream)
        return out, None, None, None, None, None


def balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, *, scoring: str = "softmax", coef: float = 1.0,
                 cu_seqlens: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """-> (loss, a fp32 scalar with a gradient to the logits; counts int32 [sequences, E] of the choice).

    Per sequence with n live tokens (those with an id; -1 is none): L = sum_e f_e P_e with f_e = E / (k n) * count_e and
    P_e the mean over the live tokens of p_te, p the row's softmax or its sigmoids normalised to sum 1; the loss is coef
    times the mean of L over the sequences that have a live token (0 without any).  1 * coef means perfect balance.
    The counts have no gradient.  ``cu_seqlens`` (int32 [S + 1] on the device, starting at 0, not decreasing) packs
    sequences; without it all tokens are one.  Tokens behind the last sequence take no part and have gradient 0.  Loss
    and gradient are the same bits every time."""
    _check_logits(logits, scoring)
    t, e = logits.shape
    if not 1 <= t <= 1 << 24:
        raise ValueError(f"need 1 to {1 << 24} tokens, got {t}")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != t or not 1 <= topk_ids.shape[1] <= min(e, MAX_TOPK):
        raise ValueError(f"topk_ids must be [{t}, k] with 1 <= k <= {min(e, MAX_TOPK)}, got {tuple(topk_ids.shape)}")
    ids = _device_int("topk_ids", topk_ids, logits, None)
    seqs = 1
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or not 2 <= cu_seqlens.numel() <= (1 << 20) + 1:
            raise ValueError(f"cu_seqlens must be [sequences + 1] of 1 to {1 << 20} sequences, got "
                             f"{tuple(cu_seqlens.shape)}")
        cu_seqlens = _device_int("cu_seqlens", cu_seqlens, logits, None)
        seqs = cu_seqlens.numel() - 1
    return _BalanceLoss.apply(logits, ids, _SCORING[scoring], float(coef), cu_seqlens, seqs)


def expert_counts(topk_ids: torch.Tensor, num_experts: int) -> torch.Tensor:
    """How often each expert occurs in topk_ids (int32 [T, k]; ids outside [0, num_experts), such as the -1 of padding,
    are skipped) -> int32 [num_experts]."""
    if topk_ids.dtype != torch.int32 or topk_ids.dim() != 2 or not topk_ids.is_cuda:
        raise ValueError(f"topk_ids must be a CUDA int32 tensor [tokens, k], got {topk_ids.dtype} "
                         f"{tuple(topk_ids.shape)} on {topk_ids.device}")
    if not 1 <= num_experts <= MAX_EXPERTS or not 1 <= topk_ids.shape[1] <= MAX_TOPK:
        raise ValueError(f"need 1 to {MAX_EXPERTS} experts and 1 to {MAX_TOPK} ids per token, got {num_experts} and "
                         f"{topk_ids.shape[1]}")
    t, k = topk_ids.shape
    if t == 0:
        return torch.zeros(num_experts, dtype=torch.int32, device=topk_ids.device)
    if t > 1 << 24:
        raise ValueError(f"at most {1 << 24} tokens, got {t}")
    ids = topk_ids.contiguous()
    counts = torch.empty(num_experts, dtype=torch.int32, device=ids.device)
    with _OnDevice(ids.get_device()) as stream:
        N.run("asap_expert_counts", ids.data_ptr(), t, k, num_experts, counts.data_ptr(), stream)
    return counts
