"""FP8 block-scaled linear and shared expert against the definition in 64 bits.

Tolerances.  A product of two E4M3 values is exact in fp32; the tensor core adds the 128 of a K block in fp32, and KB
blocks are folded with one fma each: |error| <= (128 + KB + 4) * 2^-23 * S with S = sum_k |x_k w_k| over the dequantised
values (2^-23, a whole unit, since the tensor core may truncate).  The result is rounded to its type once: eps / 2 of its
value, and 2^-25 (half of fp16's smallest step) where it is subnormal.  The input's codes are exact by definition.  In
the shared expert h carries such an error into its requantisation; there each value may take any code that its error
interval reaches, and the deviation is carried through the second product."""

import pytest
import torch

from asap_b200 import linear as lin
from asap_b200.linear import Fp8Linear, Fp8SharedExpert

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------------- the definition
def e4m3(q):
    """float64 -> the nearest E4M3 value, ties to even, saturating."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))).clamp_min(-6.0) - 3.0)
    return (torch.round(q / step) * step).clamp(-448.0, 448.0)


def blocks_of(x):
    m, k = x.shape
    out = torch.zeros(m, -(-k // 128) * 128, dtype=torch.float64, device=x.device)
    out[:, :k] = x.double()
    return out.view(m, -1, 128)


def pow2_ceil(v):
    frac, exp = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), exp - (frac == 0.5).to(exp.dtype))


def quantized_input(x, pow2):
    """What x's codes stand for: the fp32 form rounds the factor 448 / amax and the product to fp32."""
    b = blocks_of(x)
    amax = b.abs().amax(2, keepdim=True).clamp_min(torch.tensor(1e-10).item())
    if pow2:
        scale = pow2_ceil(amax / 448.0)
        q = b / scale
    else:
        scale = (amax / 448.0).float().double()
        q = (b * (448.0 / amax).float().double()).float().double()
    return (e4m3(q) * scale).view(x.shape[0], -1)[:, :x.shape[1]]


def dequantized(w, scale):
    s = scale.float().double()
    return w.double() * s.repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :w.shape[1]]


def weight(gen, n, k, scales):
    nb, kb = -(-n // 128), -(-k // 128)
    w = torch.zeros(nb * 128, kb * 128, device=DEV)
    w[:n, :k] = 0.02 * torch.randn(n, k, device=DEV, generator=gen)
    b = w.view(nb, 128, kb, 128)
    b *= torch.exp2(4.0 * torch.rand(nb, 1, kb, 1, device=DEV, generator=gen) - 2.0)
    scale = b.abs().amax((1, 3)).clamp_min(1e-12) / 448.0
    if scales == "e8m0":
        scale = pow2_ceil(scale)
    codes = (b / scale[:, None, :, None]).clamp(-448, 448).view(nb * 128, kb * 128)[:n, :k].to(torch.float8_e4m3fn)
    return codes.contiguous(), scale.to(torch.float8_e8m0fnu) if scales == "e8m0" else scale


def accumulated(x, w):
    """(x w^T, its error bound before the last rounding), float64."""
    kb = -(-x.shape[1] // 128)
    return x @ w.t(), (128 + kb + 4) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def rounding(y, dtype):
    return torch.finfo(dtype).eps / 2 * y.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check_linear(y, x, w, scale):
    ref, err = accumulated(quantized_input(x, scale.dtype != torch.float32), dequantized(w, scale))
    tol = err + rounding(ref.abs() + err, y.dtype)
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the bound, worst " \
                          f"{((y.double() - ref).abs() / tol.clamp_min(1e-300)).max().item():.2f}"


def hidden(gen, m, k, dtype):
    return (torch.randn(m, k, device=DEV, generator=gen) *
            torch.exp(0.5 * torch.randn(k, device=DEV, generator=gen))).to(dtype)


# --------------------------------------------------------------------------------------------------------- linear
SIZES = [  # m, k, n: one row, the end of the in-kernel form, each tile width, split K, the 128 x 256 tiles, ragged ends
    (1, 16, 16), (1, 128, 128), (2, 16384, 128), (3, 144, 48), (4, 7168, 256), (5, 7168, 256), (16, 512, 256),
    (17, 2064, 1040), (32, 640, 144), (33, 1024, 128), (64, 1024, 272), (65, 640, 144), (80, 512, 1040), (127, 256, 384),
    (129, 2048, 512), (130, 16384, 256), (300, 384, 272), (515, 1536, 4096), (1003, 2064, 1040), (2500, 256, 4096),
    (700, 128, 19200)]


@pytest.mark.parametrize("scales,dtype", [("fp32", torch.bfloat16), ("fp32", torch.float16), ("e8m0", torch.bfloat16),
                                          ("e8m0", torch.float16)])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_against_the_definition(cuda_ok, m, k, n, scales, dtype):
    gen = torch.Generator(device=DEV).manual_seed(m * 7 + k + n)
    w, s = weight(gen, n, k, scales)
    layer = Fp8Linear(w, s)
    x = hidden(gen, m, k, dtype)
    y = layer(x)
    lin.check()
    assert y.dtype == dtype and y.shape == (m, n)
    check_linear(y, x, w, s)
    assert torch.equal(layer(x), y), "the same call gives the same bits"


# Fewer 128 x 256 tiles than SMs and a long K: two or four CTAs share a tile's K blocks.  Whole and ragged tiles, K blocks
# that do not divide (K = 5904: 47 of them), each on two streams at once and from a replayed graph.
@pytest.mark.parametrize("scales,dtype", [("fp32", torch.bfloat16), ("fp32", torch.float16), ("e8m0", torch.bfloat16)])
@pytest.mark.parametrize("m,k,n", [(384, 7168, 4096), (333, 5904, 4080), (640, 7168, 2048), (160, 7168, 4096),
                                   (600, 7168, 1040), (601, 5904, 1040)])
def test_linear_shares_a_tile_among_ctas(cuda_ok, m, k, n, scales, dtype):
    gen = torch.Generator(device=DEV).manual_seed(m + k + n)
    w, s = weight(gen, n, k, scales)
    layer = Fp8Linear(w, s)
    x = hidden(gen, m, k, dtype)
    y = layer(x)
    lin.check()
    check_linear(y, x, w, s)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    torch.cuda.synchronize()
    for st in streams * 3:
        with torch.cuda.stream(st):
            outs.append(layer(x))
    torch.cuda.synchronize()
    wide = torch.full((m + 2, n), 7.0, dtype=dtype, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer(x, out=wide[1:m + 1])
    for _ in range(3):
        graph.replay()
    lin.check()
    assert all(torch.equal(o, y) for o in outs) and torch.equal(wide[1:m + 1], y)
    assert (wide[0] == 7).all() and (wide[m + 1] == 7).all()


@pytest.mark.parametrize("m", [3, 40, 600])
@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
def test_linear_takes_any_strides(cuda_ok, m, scales):
    gen = torch.Generator(device=DEV).manual_seed(m)
    w, s = weight(gen, 256, 272, scales)
    layer = Fp8Linear(w, s)
    wide = hidden(gen, m, 600, torch.bfloat16)
    for x in (wide[:, :272],                 # rows further apart
              wide[:, 8:280],                # 16-byte aligned, offset
              wide[:, 1:273],                # not aligned
              wide[:, :544:2],               # columns apart
              wide[:, :272].flip(0),
              hidden(gen, 272, m, torch.bfloat16).t(),
              hidden(gen, 1, 272, torch.bfloat16).expand(m, 272)):
        check_linear(layer(x), x, w, s)
    x3 = hidden(gen, 2 * m, 272, torch.bfloat16).view(2, m, 272)
    y3 = layer(x3)
    assert y3.shape == (2, m, 256)
    check_linear(y3.view(-1, 256), x3.reshape(-1, 272), w, s)
    out = torch.empty(m, 256, dtype=torch.bfloat16, device=DEV)
    assert layer(wide[:, :272], out=out) is out
    assert torch.equal(out, layer(wide[:, :272].contiguous()))
    assert layer(wide[:0, :272]).shape == (0, 256)
    assert layer(wide[0, :272].contiguous()).shape == (256,)


@pytest.mark.parametrize("m", [4, 30, 200, 700])
@pytest.mark.parametrize("scales", ["fp32", "e8m0"])
def test_linear_special_values_stay_in_their_row(cuda_ok, m, scales):
    gen = torch.Generator(device=DEV).manual_seed(m + 1)
    w, s = weight(gen, 384, 640, scales)
    layer = Fp8Linear(w, s)
    x = hidden(gen, m, 640, torch.bfloat16)
    clean = layer(x)
    x[0, 5], x[1, 639], x[2, 130] = float("nan"), float("inf"), float("-inf")
    x[3] = 0
    y = layer(x)
    assert y[:3].isnan().all() and (y[3] == 0).all()
    assert torch.equal(y[4:], clean[4:])
    x = torch.zeros(m, 640, device=DEV, dtype=torch.bfloat16)
    x[0, 0], x[1, 0], x[2, 0] = 3e38, 1e-30, -1e-38   # amax below 1e-10 counts as 1e-10: these codes are 0
    y = layer(x)
    check_linear(y[1:], x[1:], w, s)
    assert (y[1:3] == 0).all() and not y[0].isnan().any()


@pytest.mark.parametrize("m", [1, 40, 300, 1200])
def test_linear_streams_and_graphs(cuda_ok, m):
    """Two streams at once, and two graphs of one layer replayed in turn and at the same time, share nothing."""
    gen = torch.Generator(device=DEV).manual_seed(m)
    w, s = weight(gen, 512, 1024, "fp32")
    layer = Fp8Linear(w, s)
    xs = [hidden(gen, m, 1024, torch.bfloat16) for _ in range(4)]
    want = [layer(x) for x in xs]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = [None] * 4
    for i in range(4):
        with torch.cuda.stream((a, b)[i % 2]):
            for _ in range(5):
                got[i] = layer(xs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    graphs, outs, ins = [], [], [x.clone() for x in xs[:2]]
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(x))
        graphs.append(g)
    for i in (0, 1):
        ins[i].copy_(xs[2 + i])
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[2]) and torch.equal(outs[1], want[3])
    lin.check()


FIRST_CALL_CAPTURED = """
import torch
from asap_b200.linear import Fp8Linear, Fp8SharedExpert
from asap_b200.router import balance_loss, expert_counts, route
gen = torch.Generator(device="cuda").manual_seed(0)
w = 0.02 * torch.randn(256, 256, device="cuda", generator=gen)
layer = Fp8Linear.from_float(w)
shared = Fp8SharedExpert.from_float(w, 0.02 * torch.randn(256, 128, device="cuda", generator=gen))
x = torch.randn({m}, 256, device="cuda", generator=gen).bfloat16()
torch.cuda.synchronize()
def run():
    y = layer(x)
    top = route(y, 8, scoring="sigmoid", bias=w[0])
    loss, counts = balance_loss(y, top.topk_ids, scoring="sigmoid")
    return y, shared(x), top.topk_weights, top.topk_ids, loss, counts, expert_counts(top.topk_ids, 256)
g = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(g):
    got = run()
g.replay()
torch.cuda.synchronize()
with torch.no_grad():
    want = run()
assert all(torch.equal(a, b) for a, b in zip(got, want))
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        Fp8Linear.from_float(w)
except RuntimeError as e:
    assert "being captured" in str(e), e
else:
    raise AssertionError("a layer was made in a capture")
print("captured first")
"""


@pytest.mark.parametrize("m", [2, 600])
def test_first_calls_of_a_process_may_be_captured(cuda_ok, m):
    import os
    import subprocess
    import sys

    env = dict(os.environ, PYTHONPATH=os.pathsep.join(sys.path))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED.replace("{m}", str(m))], env=env, capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_linear_from_float_and_release(cuda_ok):
    gen = torch.Generator(device=DEV).manual_seed(0)
    layer = Fp8Linear.from_float(0.02 * torch.randn(256, 384, device=DEV, generator=gen))
    assert layer.shape == (256, 384)
    x = hidden(gen, 20, 384, torch.bfloat16)
    check_linear(layer(x), x, layer._w.w.view(torch.float8_e4m3fn), layer._w.scale)
    layer.release()
    layer.release()
    with pytest.raises(RuntimeError, match="released"):
        layer(x)


def test_linear_refusals(cuda_ok):
    gen = torch.Generator(device=DEV).manual_seed(0)
    w, s = weight(gen, 128, 256, "fp32")
    layer = Fp8Linear(w, s)
    x = hidden(gen, 4, 256, torch.bfloat16)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        layer(x.float())
    with pytest.raises(ValueError, match="x must be"):
        layer(x[:, :128])
    with pytest.raises(ValueError, match="x must be"):
        layer(x.cpu())
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(x.clone().requires_grad_(True))
    with torch.no_grad():
        layer(x.clone().requires_grad_(True))
    for out in (torch.empty(4, 128, device=DEV), torch.empty(5, 128, device=DEV, dtype=torch.bfloat16),
                torch.empty(128, 4, device=DEV, dtype=torch.bfloat16).t()):
        with pytest.raises(ValueError, match="out must be"):
            layer(x, out=out)
    buf = torch.empty(4 * 256 + 4 * 128, device=DEV, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share memory"):
        layer(buf[:1024].view(4, 256), out=buf[512:1024].view(4, 128))
    layer(buf[:1024].view(4, 256).zero_(), out=buf[1024:].view(4, 128))
    with pytest.raises(ValueError, match="scales of shape"):
        Fp8Linear(w, s[:, :1])
    with pytest.raises(ValueError, match="scales of shape"):
        Fp8Linear(w, s.half())
    with pytest.raises(ValueError, match="multiples of 16"):
        Fp8Linear(w[:, :24].contiguous(), s[:, :1].contiguous())
    with pytest.raises(ValueError, match="contiguous E4M3"):
        Fp8Linear(w.view(torch.uint8).t(), s)
    with pytest.raises(ValueError, match="one CUDA device"):
        Fp8Linear(w.cpu(), s.cpu())


# --------------------------------------------------------------------------------------------------- shared expert
def quantized_h(h, dh, pow2):
    """(what h's codes stand for, how far the codes of any h within dh can be from that)."""
    b, d = blocks_of(h), blocks_of(dh)
    amax = b.abs().amax(2, keepdim=True)
    slack = d.amax(2, keepdim=True)

    def values(v, a):
        a = a.clamp_min(1e-10)
        scale = pow2_ceil(a / 448.0) if pow2 else a / 448.0
        return e4m3(v / scale) * scale
    ref = values(b, amax)
    dev = torch.zeros_like(ref)
    for v in (b - d, b + d):
        for a in (amax - slack, amax + slack):
            dev = torch.maximum(dev, (values(v, a) - ref).abs())
    dev = dev + 2.0 ** -22 * ref.abs()  # the fp32 scale and factor
    return ref.view(h.shape[0], -1)[:, :h.shape[1]], dev.view(h.shape[0], -1)[:, :h.shape[1]]


@pytest.mark.parametrize("scales,dtype,limit", [("fp32", torch.bfloat16, 0.0), ("fp32", torch.float16, 0.75),
                                                ("e8m0", torch.bfloat16, 0.75), ("e8m0", torch.float16, 0.0)])
@pytest.mark.parametrize("m,hidden_size,inter", [(1, 7168, 256), (4, 1024, 512), (17, 2064, 128), (40, 1024, 384),
                                                 (65, 512, 256), (200, 1024, 512), (1000, 1024, 512),
                                                 (2100, 256, 1280)])
def test_shared_expert_against_the_definition(cuda_ok, m, hidden_size, inter, scales, dtype, limit):
    gen = torch.Generator(device=DEV).manual_seed(m + hidden_size)
    w13, s13 = weight(gen, 2 * inter, hidden_size, scales)
    w2, s2 = weight(gen, hidden_size, inter, scales)
    layer = Fp8SharedExpert(w13, s13, w2, s2, swiglu_limit=limit)
    x = hidden(gen, m, hidden_size, dtype)
    y = layer(x)
    lin.check()
    pow2 = scales == "e8m0"
    gu, err = accumulated(quantized_input(x, pow2), dequantized(w13, s13))
    (g, u), (eg, eu) = gu.split(inter, 1), err.split(inter, 1)
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    silu = g * torch.sigmoid(g)
    h = silu * u
    # |silu'| <= 1.1; expf, the sum, the division and the products round 8 times
    dh = 1.1 * u.abs() * eg + (silu.abs() + 1.1 * eg) * eu + 8 * 2.0 ** -23 * h.abs()
    q, dq = quantized_h(h, dh, pow2)
    wd = dequantized(w2, s2)
    ref, acc = accumulated(q, wd)
    tol = acc + dq @ wd.abs().t()
    tol = tol + rounding(ref.abs() + tol, dtype)
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the bound"
    # the bound must not be empty talk: the result is close in the norm as well, to a few roundings of its type and h's
    rel = ((y.double() - ref).norm() / ref.norm()).item()
    assert rel < torch.finfo(dtype).eps / 2 + 2.0 ** -9, rel
    assert torch.equal(layer(x), y)


def test_shared_expert_special_rows_out_and_refusals(cuda_ok):
    gen = torch.Generator(device=DEV).manual_seed(5)
    w13, s13 = weight(gen, 512, 384, "fp32")
    w2, s2 = weight(gen, 384, 256, "fp32")
    layer = Fp8SharedExpert(w13, s13, w2, s2)
    for m in (6, 900):
        x = hidden(gen, m, 384, torch.bfloat16)
        clean = layer(x)
        x[0, 1], x[1, 2] = float("nan"), float("inf")
        x[2] = 0
        out = torch.full_like(clean, 7.0)
        assert layer(x, out=out) is out
        assert out[:2].isnan().all() and (out[2] == 0).all() and torch.equal(out[3:], clean[3:])
    assert layer(x[:0]).shape == (0, 384)
    e13, t13 = weight(gen, 512, 384, "e8m0")
    with pytest.raises(ValueError, match="one kind of scales"):
        Fp8SharedExpert(e13, t13, w2, s2)
    with pytest.raises(ValueError, match=r"need w13 \[2I, H\]"):
        Fp8SharedExpert(w13, s13, w13, s13)
    with pytest.raises(RuntimeError, match="no gradient"):
        layer(hidden(gen, 4, 384, torch.bfloat16).requires_grad_(True))
