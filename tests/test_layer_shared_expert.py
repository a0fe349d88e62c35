"""AsapMoE.forward with a shared expert that raises: the dispatched message is still combined (with the channel replaced by
a recorder, no GPU)."""

import pytest
import torch

from asap_b200.dispatcher import AsapBuffer
from asap_b200.layer import AsapMoE
from asap_b200.sglang_shim import StandardTopKOutput


class Buffer:
    n_max = 8

    def __init__(self):
        self.sent, self.received, self.fail = [], [], None

    def send(self, layer_id, x, ids, weights, micro_batch=None):
        self.sent.append(len(self.sent))
        return self.sent[-1], (x, ids, weights)

    def recv(self, ticket, shared=None):
        if self.fail is not None:
            raise self.fail
        if shared is not None and shared.dtype != torch.bfloat16:
            raise TypeError("shared must be bf16 [n_tokens, hidden]")
        self.received.append(ticket)
        return torch.zeros(4, 16, dtype=torch.bfloat16) if shared is None else shared

    def exchange(self, layer_id, x, ids, weights):
        return torch.zeros_like(x)


@pytest.fixture
def buffer():
    buffer, old = Buffer(), AsapBuffer._buffer
    AsapBuffer.install(buffer)
    yield buffer
    AsapBuffer.install(old)


def layer_with(shared):
    layer = AsapMoE(num_experts=8, hidden_size=16, intermediate_size=16, layer_id=0, top_k=2)
    layer.shared_expert = shared
    return layer


def inputs(n=4):
    return (torch.ones(n, 16, dtype=torch.bfloat16),
            StandardTopKOutput(torch.ones(n, 2), torch.zeros(n, 2, dtype=torch.int32), None))


def test_a_shared_expert_that_raises_leaves_no_message_behind(buffer):
    def refuses(x):
        assert buffer.sent and not buffer.received  # it runs while the F ranks work
        raise ValueError("x must be something else")

    with pytest.raises(ValueError, match="something else"):
        layer_with(refuses)(*inputs())
    assert buffer.sent == buffer.received == [0]
    out = layer_with(lambda x: 2 * x)(*inputs())
    assert buffer.sent == buffer.received == [0, 1] and (out == 2).all()


def test_a_shared_output_of_another_type_leaves_no_message_behind(buffer):
    with pytest.raises(TypeError, match="bf16"):
        layer_with(lambda x: x.float())(*inputs())
    assert buffer.sent == buffer.received == [0]


def test_the_first_error_is_the_one_that_is_raised(buffer):
    def refuses(x):
        buffer.fail = RuntimeError("the channel is poisoned")
        raise ValueError("the expert's own")

    with pytest.raises(ValueError, match="own"):
        layer_with(refuses)(*inputs())


def test_nothing_to_take_back_when_nothing_is_in_flight(buffer):
    def refuses(x):
        raise ValueError("no")

    for n in (0, 20):  # an empty batch; one that was exchanged in pieces
        with pytest.raises(ValueError, match="no"):
            layer_with(refuses)(*inputs(n))
    assert buffer.sent == buffer.received == []
