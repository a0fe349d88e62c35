"""Who hears of a wait that a kernel of the FP8 products gave up: the next call, the channel's check, linear.check.  The
report is written here by the host, in place of a kernel's."""

import ctypes

import pytest
import torch

from asap_b200 import _native as N
from asap_b200 import linear
from asap_b200.transport.channel import AttnChannel
from asap_b200.transport.layout import Geometry

WORD = 5  # pipeline timeout


class Word(linear._Status):
    def __init__(self):
        self.word, self.ptr = ctypes.c_uint64(0), 0


@pytest.fixture
def two(monkeypatch):
    words, waited = {0: Word(), 1: Word()}, []
    monkeypatch.setattr(linear, "_status", words)
    monkeypatch.setattr(torch.cuda, "synchronize", waited.append)
    return words, waited


def test_check_asks_every_device_unless_told_which(two):
    words, waited = two
    linear.check()
    assert waited == [0, 1]
    words[1].word.value = WORD
    linear.check(0)
    with pytest.raises(N.AsapError, match="gave up a wait"):
        linear.check()
    linear.check()  # said once
    words[1].word.value = WORD
    with pytest.raises(N.AsapError, match="gave up a wait"):
        linear.check(1)


def test_poll_waits_for_nothing(two):
    words, waited = two
    linear.poll()
    words[0].word.value = WORD
    linear.poll(1)
    with pytest.raises(N.AsapError):
        linear.poll(0)
    assert waited == []


def test_the_channel_of_that_device_raises(two):
    words, _ = two
    channel = AttnChannel(0, Geometry(1, 1, 1, 64, 256, 2, 1), [("127.0.0.1", 1)], device=1)
    channel.check()
    words[0].word.value = WORD
    channel.check()  # another device's
    words[1].word.value = WORD
    with pytest.raises(N.AsapError, match="gave up a wait"):
        channel.check()
    channel.check()


def test_the_next_call_of_a_layer_raises(two):
    words, _ = two

    class Weight:  # what a registered weight looks like to the checks of a call
        handle, reports, k = 1, words[0], 256

    words[0].word.value = WORD
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(N.AsapError, match="gave up a wait"):
        linear._rows(x, Weight, None, 128)
    assert words[0].word.value == 0
