"""What the C entry points of the linear, the router and the balance loss refuse without touching a GPU, and what the
Python layer refuses of CPU tensors."""

import ctypes

import pytest
import torch

from asap_b200 import _native as N
from asap_b200 import router
from asap_b200.linear import Fp8Linear


def err() -> str:
    return N.lib().asap_last_error_string().decode()


@pytest.mark.parametrize("n,k", [(0, 128), (128, 0), (120, 128), (128, 24), (1 << 18, 128), (-16, 16)])
def test_linear_register_refuses_shapes(n, k):
    d, h = N.Fp8Linear_t(n, k, 4096, 4096, 0), ctypes.c_uint64()
    assert N.lib().asap_fp8_linear_register(ctypes.byref(d), ctypes.byref(h)) == N.ASAP_EINVAL
    assert "multiples of 16" in err()


@pytest.mark.parametrize("w,scale,atoms", [(0, 4096, 0), (4104, 4096, 0), (4096, 0, 0), (4096, 4098, 0), (4096, 4096, 8)])
def test_linear_register_refuses_pointers(w, scale, atoms):
    d, h = N.Fp8Linear_t(128, 128, w, scale, atoms), ctypes.c_uint64()
    assert N.lib().asap_fp8_linear_register(ctypes.byref(d), ctypes.byref(h)) == N.ASAP_EINVAL
    assert "aligned" in err()
    assert N.lib().asap_fp8_linear_register(None, ctypes.byref(h)) == N.ASAP_EINVAL


def test_linear_calls_refuse_unknown_handles():
    lib = N.lib()
    assert lib.asap_fp8_linear(987654, 4096, 128, 4, 0, 4096, 4096, 1 << 20, 0, 1, None) == N.ASAP_EINVAL
    assert "unknown handle" in err()
    assert lib.asap_fp8_shared(987654, 987655, 4096, 128, 4, 0, 0.0, 4096, 4096, 1 << 20, 0, 1, None) == N.ASAP_EINVAL
    assert lib.asap_fp8_linear_release(987654) == N.ASAP_EINVAL


def test_workspace_sizes():
    lib = N.lib()
    assert lib.asap_fp8_linear_ws_bytes(0, 128) == 0 and lib.asap_fp8_linear_ws_bytes(5, 0) == 0
    assert lib.asap_fp8_linear_ws_bytes(1, 7168) == 0  # one launch, no scratch
    # codes [m, k] and a scale per row (to 128) and block
    assert lib.asap_fp8_linear_ws_bytes(1000, 7168) >= 1000 * 7168 + 1024 * 56 * 4
    assert lib.asap_fp8_linear_ws_bytes(1000, 2064) >= 1000 * 17 * 128 + 1024 * 17 * 4
    assert lib.asap_fp8_shared_ws_bytes(4, 1024, 512) >= 4 * 1536 + 128 * 12 * 4
    assert lib.asap_fp8_shared_ws_bytes(0, 1024, 512) == 0
    assert lib.asap_balance_ws_bytes(0, 1) == 0 and lib.asap_balance_ws_bytes(4, 0) == 0
    assert lib.asap_balance_ws_bytes(1000, 7) >= 4 * 1000 + 8 * 7


def route_desc(**kw):
    v = dict(logits=4096, ld=64, dtype=0, t=4, e=64, k=2, sigmoid=0, groups=1, top_groups=1, renormalize=1, scale=1.0,
             pad=0, bias=0, num_tokens=0)
    v.update(kw)
    return N.Route_t(*[v[n] for n, _ in N.Route_t._fields_])


@pytest.mark.parametrize("kw", [dict(t=0), dict(e=0), dict(e=1025, ld=1025), dict(k=0), dict(k=33), dict(k=65), dict(ld=63),
                                dict(dtype=3), dict(logits=0), dict(logits=4098), dict(groups=3), dict(groups=64),
                                dict(groups=8, top_groups=9), dict(top_groups=0), dict(bias=4097), dict(num_tokens=2)])
def test_route_refuses(kw):
    d = route_desc(**kw)
    assert N.lib().asap_route(ctypes.byref(d), 4096, 4096, None) == N.ASAP_EINVAL
    assert N.lib().asap_route(None, 4096, 4096, None) == N.ASAP_EINVAL


def test_route_refuses_results():
    d = route_desc()
    for ids, w in ((0, 4096), (4096, 0), (4097, 4096)):
        assert N.lib().asap_route(ctypes.byref(d), ids, w, None) == N.ASAP_EINVAL
    for args in ((0, 4096, 4096), (4096, 0, 4096), (4096, 4096, 0)):
        assert N.lib().asap_route_backward(ctypes.byref(d), *args, None) == N.ASAP_EINVAL


def balance_desc(**kw):
    v = dict(logits=4096, ld=64, dtype=1, t=4, e=64, k=2, sigmoid=1, seqs=1, coef=1.0, pad=0, ids=4096, cu_seqlens=0,
             counts=4096)
    v.update(kw)
    return N.Balance_t(*[v[n] for n, _ in N.Balance_t._fields_])


@pytest.mark.parametrize("kw", [dict(t=0), dict(e=2000, ld=2000), dict(k=0), dict(ld=3), dict(ids=0), dict(counts=0),
                                dict(seqs=0), dict(seqs=2), dict(cu_seqlens=6), dict(logits=4097)])
def test_balance_refuses(kw):
    d = balance_desc(**kw)
    n = 1 << 20
    assert N.lib().asap_balance_loss(ctypes.byref(d), 4096, n, 4096, None) == N.ASAP_EINVAL
    assert N.lib().asap_balance_backward(ctypes.byref(d), 4096, n, 4096, 4096, None) == N.ASAP_EINVAL


def test_balance_and_counts_refuse_buffers():
    lib, d = N.lib(), balance_desc()
    need = lib.asap_balance_ws_bytes(4, 1)
    assert lib.asap_balance_loss(ctypes.byref(d), 4096, need - 1, 4096, None) == N.ASAP_EINVAL
    assert lib.asap_balance_loss(ctypes.byref(d), 4100, need, 4096, None) == N.ASAP_EINVAL
    assert lib.asap_balance_loss(ctypes.byref(d), 4096, need, 0, None) == N.ASAP_EINVAL
    assert lib.asap_balance_backward(ctypes.byref(d), 4096, need, 0, 4096, None) == N.ASAP_EINVAL
    for args in ((0, 4, 2, 8, 4096), (4096, 0, 2, 8, 4096), (4096, 4, 33, 8, 4096), (4096, 4, 2, 1025, 4096),
                 (4096, 4, 2, 8, 0)):
        assert lib.asap_expert_counts(*args, None) == N.ASAP_EINVAL


def test_python_refuses_cpu_tensors_and_values():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        router.route(x, 2)
    with pytest.raises(ValueError, match="CUDA"):
        router.balance_loss(x, torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        router.expert_counts(torch.zeros(4, 2, dtype=torch.int32), 8)
    with pytest.raises(ValueError, match="one CUDA device"):
        Fp8Linear(torch.zeros(128, 128, dtype=torch.uint8), torch.ones(1, 1))
    with pytest.raises(ValueError, match="multiples of 16"):
        Fp8Linear(torch.zeros(120, 128, dtype=torch.uint8), torch.ones(1, 1))
