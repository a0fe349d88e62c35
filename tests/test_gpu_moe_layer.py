"""One MoE layer of an attention rank as a whole: the router's choice goes to the dispatch, the FP8 shared expert runs
while the F rank works, the combine adds both; against the oracle, relative L2 1e-2 of the reference semantics with the
same activation quantisation.  Then the same from a captured router, and with experts switched off."""

import numpy as np
import pytest
import torch

from asap_b200.experts import Fp8Experts
from asap_b200.layer import AsapMoE
from asap_b200.linear import Fp8Linear, Fp8SharedExpert
from asap_b200.loopback import Loopback
from asap_b200.router import balance_loss, expert_counts, route
from asap_b200.transport.layout import Geometry
from gpu_util import experts_to_oracle, np_from_bf16
from oracle import moe, mx

pytestmark = pytest.mark.gpu
E, H, I, K = 16, 1024, 512, 4


@pytest.fixture(scope="module")
def layer(cuda_ok):
    experts = Fp8Experts.random(E, H, I, seed=3)
    lb = Loopback(Geometry(1, 1, 2, 512, H, K, 1), {2: experts}, timeout_s=5.0)
    lb.install()
    gen = torch.Generator(device="cuda").manual_seed(1)
    moe_layer = AsapMoE(E, H, I, 2, top_k=K)
    moe_layer.shared_expert = Fp8SharedExpert.from_float(0.02 * torch.randn(2 * I, H, device="cuda", generator=gen),
                                                         0.02 * torch.randn(H, I, device="cuda", generator=gen))
    gate = Fp8Linear.from_float(0.05 * torch.randn(128, H, device="cuda", generator=gen))
    yield lb, moe_layer, gate, experts_to_oracle(experts)
    lb.close()
    experts.release()


def shared_oracle(x, s):
    w13 = mx.fp8_block_dequantize(s._w13.w.cpu().numpy(), s._w13.scale.cpu().numpy())
    w2 = mx.fp8_block_dequantize(s._w2.w.cpu().numpy(), s._w2.scale.cpu().numpy())
    gu = mx.fp8_act_roundtrip(x).astype(np.float64) @ w13.T.astype(np.float64)
    h = moe.silu(gu[:, :I].astype(np.float32)) * gu[:, I:].astype(np.float32)
    return mx.fp8_act_roundtrip(h.astype(np.float32)) @ w2.T


@pytest.mark.parametrize("T", [1, 7, 130, 512, 700])  # 700: more than a message, sent in pieces
def test_layer_with_router_and_shared_expert(layer, T):
    lb, moe_layer, gate, (w_gate, w_up, w_down) = layer
    gen = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, H, device="cuda", generator=gen).bfloat16()
    bias = 0.05 * torch.randn(E, device="cuda", generator=gen)
    with torch.no_grad():
        logits = gate(x)[:, :E]  # a column slice of the gate's product
        topk = route(logits, K, scoring="sigmoid", bias=bias, num_groups=4, top_groups=2, routed_scaling_factor=2.5)
        out = moe_layer(x, topk)
    torch.cuda.synchronize()
    lb.check()
    ids, w, xs = topk.topk_ids.cpu().numpy(), topk.topk_weights.cpu().numpy(), np_from_bf16(x)
    assert (ids >= 0).all() and np.allclose(w.sum(1), 2.5, rtol=1e-5)
    ref = moe.ffn_rank(xs, ids, w, w_gate, w_up, w_down, 0, E, act_quant="fp8") + shared_oracle(xs, moe_layer.shared_expert)
    assert moe.rel_l2(np_from_bf16(out), ref) < 1e-2
    np.testing.assert_array_equal(expert_counts(topk.topk_ids, E).cpu().numpy(), np.bincount(ids.ravel(), minlength=E))
    loss, counts = balance_loss(logits, topk.topk_ids, scoring="sigmoid")
    np.testing.assert_array_equal(counts[0].cpu().numpy(), np.bincount(ids.ravel(), minlength=E))
    assert loss.item() > 0


def test_padded_batch_and_switched_off_experts(layer):
    """Rows behind the valid tokens dispatch nothing and come back as their shared expert alone; experts switched off
    by -inf get no token."""
    lb, moe_layer, gate, (w_gate, w_up, w_down) = layer
    T, n = 96, 61
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(T, H, device="cuda", generator=gen).bfloat16()
    with torch.no_grad():
        logits = gate(x)[:, :E].clone()
        logits[:, 8:] = float("-inf")
        topk = route(logits, K, num_tokens=torch.tensor([n], dtype=torch.int32, device="cuda"))
        out = moe_layer(x, topk)
        shared = moe_layer.shared_expert(x)
    torch.cuda.synchronize()
    lb.check()
    counts = expert_counts(topk.topk_ids, E)
    assert counts[8:].sum() == 0 and counts[:8].sum() == n * K
    assert torch.equal(out[n:], shared[n:])
    ids, w, xs = topk.topk_ids.cpu().numpy(), topk.topk_weights.cpu().numpy(), np_from_bf16(x)
    ref = moe.ffn_rank(xs, ids, w, w_gate, w_up, w_down, 0, E, act_quant="fp8") + shared_oracle(xs, moe_layer.shared_expert)
    assert moe.rel_l2(np_from_bf16(out), ref) < 1e-2


def test_layer_without_a_shared_expert_is_as_before(layer):
    lb, moe_layer, gate, _ = layer
    x = torch.randn(40, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    with torch.no_grad():
        topk = route(gate(x)[:, :E], K)
        plain = AsapMoE(E, H, I, 2, top_k=K)
        routed = plain(x, topk)
        both = moe_layer(x, topk)
        shared = moe_layer.shared_expert(x)
    torch.cuda.synchronize()
    lb.check()
    assert torch.equal((routed.float() + shared.float()).bfloat16(), both)
