"""The dense FP8 products of an attention rank: a linear layer over block-scaled weights, and the shared expert.

The checkpoints whose routed experts ``experts.Fp8Experts`` serves hold their dense weights in the same format: E4M3
values with one scale per 128 x 128 block.  ``Fp8Linear`` multiplies by such a weight without widening it;
``Fp8SharedExpert`` is the SwiGLU expert every token passes through, whose output the combine adds
(``AsapDispatcher.combine(out, shared=...)``, ``AsapMoE.shared_expert``; the reference adds the shared output in
python/sgl_asap_plugin/srt/batch_overlap/operations_strategy.py:106-111).

    y[r, n] = sum_b sa[r, b] * sb[n // 128, b] * sum_{k in block b} xq[r, k] * w[n, k]

Activations are quantised inside the call, per row and block b of 128 values along K:

* fp32 weight scales: sa = amax / 448, xq = e4m3(x * (448 / amax)), the quotients and the product each rounded to fp32
  (the rule of the routed experts' activations);
* E8M0 weight scales (``torch.float8_e8m0fnu``): sa = amax / 448 rounded up to a power of two, xq = e4m3(x / sa).

amax counts as at least 1e-10.  A NaN or infinity in a row makes that row of the result NaN and no other.  Sums are
held in fp32 and rounded once to x's type.  Both are for serving: they have no gradient.

A layer reads the weight tensor it was made of where it is and may hold its scales as a copy: after writing new values
into them call ``reload``.  A call allocates its scratch from torch's caching allocator on the current stream, so calls on
different streams and captured graphs share nothing.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native as N

MAX_ROWS = 1 << 20
TIMEOUT_NS = 5_000_000_000  # what the waits inside the kernels have, counted from their start


class _Status:
    """A word of pinned host memory in which a kernel reports that it gave up a wait: the host reads it with a plain
    load."""

    def __init__(self):
        self.tensor = torch.zeros(1, dtype=torch.int64, pin_memory=True)
        self.word = ctypes.c_uint64.from_address(self.tensor.data_ptr())
        self.ptr = self.tensor.data_ptr()

    def check(self) -> None:
        value = self.word.value
        if value:
            self.word.value = 0
            raise N.AsapError("asap_fp8_linear", N.ASAP_ETIMEOUT, f"a kernel gave up a wait and its call's result is "
                              f"garbage; device status {N.decode_status(value)}")


_status: dict = {}  # device index -> _Status


def _status_of(device: torch.device) -> _Status:
    status = _status.get(device.index)
    if status is None:
        status = _status[device.index] = _Status()
    return status


def poll(device: Optional[int] = None) -> None:
    """Raise if a kernel of this module has reported by now that it gave up a wait on ``device`` (None: on any).  Does
    not wait for kernels under way.  Every later call of a layer on that device does the same, and so does
    ``AttnChannel.check``, which the round trip calls for every message."""
    for index, status in list(_status.items()):
        if device is None or index == device:
            status.check()


def check(device: Optional[int] = None) -> None:
    """``poll`` after everything enqueued on ``device`` (None: on every device that has a layer) has run."""
    for index in list(_status):
        if device is None or index == device:
            torch.cuda.synchronize(index)
    poll(device)


def _scale_atoms(scale: torch.Tensor) -> torch.Tensor:
    """E8M0 scales [nb, kb] -> uint8 [kb, nb rounded up to even, 512], each byte 512 times (1/32 of the weight)."""
    b = scale.view(torch.uint8)
    nb, kb = b.shape
    atoms = torch.zeros((kb, nb + nb % 2, 512), dtype=torch.uint8, device=b.device)
    atoms[:, :nb] = b.t()[:, :, None]
    return atoms


class _Weight:
    """A registered [n, k] weight (keeps its tensors alive)."""

    def __init__(self, name: str, w: torch.Tensor, scale: torch.Tensor):
        if w.dtype == torch.float8_e4m3fn:
            w = w.view(torch.uint8)
        if w.dtype != torch.uint8 or w.dim() != 2 or not w.is_contiguous():
            raise ValueError(f"{name}: need contiguous E4M3 values [n, k] (float8_e4m3fn or their bytes), got "
                             f"{w.dtype} {tuple(w.shape)}")
        self.n, self.k = w.shape
        if self.n < 16 or self.k < 16 or self.n % 16 or self.k % 16:
            raise ValueError(f"{name}: n and k must be multiples of 16, got {self.n} x {self.k}")
        blocks = (-(-self.n // 128), -(-self.k // 128))
        if scale.dtype not in (torch.float32, torch.float8_e8m0fnu) or tuple(scale.shape) != blocks:
            raise ValueError(f"{name}: need float32 or float8_e8m0fnu scales of shape {blocks}, got {scale.dtype} "
                             f"{tuple(scale.shape)}")
        if not w.is_cuda or scale.device != w.device:
            raise ValueError(f"{name}: the weight and its scales must be on one CUDA device")
        if w.data_ptr() % 16:
            raise ValueError(f"{name}: the weight must be 16-byte aligned")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"{name}: a layer cannot be made while a CUDA graph is being captured")
        self.pow2 = scale.dtype == torch.float8_e8m0fnu
        w, scale = w.detach(), scale.detach()  # parameters may require a gradient; the layer has none
        self.w, self.given, self.scale = w, scale, scale.float().contiguous()  # scale: given's memory, or a copy
        self.device = w.device
        self.atoms = _scale_atoms(scale) if self.pow2 else None
        # what was laid out here, or by from_float, may be read on any stream from now on
        torch.cuda.current_stream(self.device).synchronize()
        self.reports = _status_of(self.device)
        self.status = self.reports.ptr
        self.handle = 0
        desc = N.Fp8Linear_t(self.n, self.k, self.w.data_ptr(), self.scale.data_ptr(),
                             self.atoms.data_ptr() if self.pow2 else 0)
        h = ctypes.c_uint64()
        with torch.cuda.device(self.device):
            N.call("asap_fp8_linear_register", ctypes.byref(desc), ctypes.byref(h))
        self.handle = h.value

    def reload(self) -> None:
        if self.scale.data_ptr() != self.given.data_ptr():
            self.scale.copy_(self.given)
        if self.pow2:
            self.atoms.copy_(_scale_atoms(self.given))

    def release(self) -> None:
        if self.handle:
            handle, self.handle = self.handle, 0
            N.call("asap_fp8_linear_release", handle)

    def __del__(self):
        try:
            self.release()
        except Exception:  # noqa: BLE001  (interpreter shutdown)
            pass


def _has_tangent(x: torch.Tensor) -> bool:
    """Forward-mode differentiation: the kernels would drop the tangent without a word."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


def _overlap(out: torch.Tensor, rows: torch.Tensor, ld: int, m: int, k: int) -> bool:
    lo, hi = rows.data_ptr(), rows.data_ptr() + 2 * ((m - 1) * ld + k)
    return m > 0 and out.data_ptr() < hi and lo < out.data_ptr() + out.numel() * out.element_size()


def _rows(x: torch.Tensor, weight: _Weight, out: Optional[torch.Tensor], n: int):
    """-> (x as rows the kernels can read, their stride, out of x's leading shape)."""
    if not weight.handle:
        raise RuntimeError("the layer was released")
    if weight.reports.word.value:
        weight.reports.check()
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] != weight.k or x.get_device() != weight.device.index:
        raise ValueError(f"x must be [..., {weight.k}] on {weight.device}, got {tuple(x.shape)} on {x.device}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("the FP8 products have no gradient: call them under torch.no_grad() or detach x")
    if _has_tangent(x):
        raise RuntimeError("the FP8 products have no forward-mode gradient: detach x")
    shape = (*x.shape[:-1], n)
    rows = x if x.dim() == 2 else x.reshape(-1, weight.k)
    m, ld = rows.shape[0], weight.k
    if m > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows per call, got {m}")
    if m > 1 and not rows.is_contiguous():
        ld = rows.stride(0)
    if rows.stride(1) != 1 or ld % 8 or ld < weight.k or rows.data_ptr() % 16:
        rows, ld = rows.clone(memory_format=torch.contiguous_format), weight.k
    if out is None:
        out = x.new_empty(shape)
    elif _overlap(out, rows, ld, m, weight.k):
        raise ValueError("out must not share memory with x")
    elif (out.dtype != x.dtype or tuple(out.shape) != shape or out.device != x.device or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError(f"out must be a contiguous, 16-byte aligned {x.dtype} tensor of shape {shape} on {x.device}")
    return rows, ld, out


class _OnDevice:
    """torch.cuda.device(index), entered only when that is not the current device, -> the device's current
    raw stream."""

    __slots__ = ("index", "prev")

    def __init__(self, index: int):
        self.index, self.prev = index, -1

    def __enter__(self) -> int:
        current = torch.cuda.current_device()
        if current != self.index:
            self.prev = current
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.prev >= 0:
            torch.cuda.set_device(self.prev)
        return False


def _scratch(nbytes: int, device: torch.device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


class Fp8Linear:
    """y = x W^T over an E4M3 weight [n, k] with one scale per 128 x 128 block, [ceil(n/128), ceil(k/128)], fp32 or
    E8M0.  n and k are multiples of 16.  x: bf16 or fp16 [..., k] of any strides -> [..., n] of its type; ``out`` takes
    the result in place of a new tensor."""

    def __init__(self, weight: torch.Tensor, scale: torch.Tensor):
        self._w = _Weight("weight", weight, scale)

    @property
    def shape(self) -> tuple:
        return self._w.n, self._w.k

    @classmethod
    def from_float(cls, w: torch.Tensor) -> "Fp8Linear":
        """A dense CUDA weight [n, k] (multiples of 128) -> block-quantised (``quant.fp8_block_quantize``)."""
        from .quant import fp8_block_quantize

        return cls(*fp8_block_quantize(w))

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        w = self._w
        rows, ld, out = _rows(x, w, out, w.n)
        m = rows.shape[0]
        if m:
            nbytes = N.lib().asap_fp8_linear_ws_bytes(m, w.k)
            ws = _scratch(nbytes, w.device)
            with _OnDevice(w.device.index) as stream:
                N.run("asap_fp8_linear", w.handle, rows.data_ptr(), ld, m, x.dtype == torch.float16, out.data_ptr(),
                      ws.data_ptr() if nbytes else 0, nbytes, w.status, TIMEOUT_NS, stream)
        return out

    def reload(self) -> None:
        """To be called after new values were written into the weight and scale tensors this layer was made of: the weight
        is read where it is, and so are contiguous fp32 scales, but of others the layer holds copies.  Renewed in place on
        the current stream, so that captured graphs see them too."""
        self._w.reload()

    def release(self) -> None:
        self._w.release()


class Fp8SharedExpert:
    """out = (silu(g) * u) W2^T with [g, u] = x W13^T: w13 [2I, H] (gate rows, then up rows), w2 [H, I], both with
    block scales as ``Fp8Linear`` takes them, of one kind; I a multiple of 128, H of 16.  ``swiglu_limit`` > 0 clamps g
    to at most and u to +-that value.  h = silu(g) * u goes to the second product requantised per row and 128 values,
    never through 16 bits."""

    def __init__(self, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor, *,
                 swiglu_limit: float = 0.0):
        self._w13, self._w2 = _Weight("w13", w13, w13_scale), _Weight("w2", w2, w2_scale)
        self.hidden, self.inter, self.swiglu_limit = self._w13.k, self._w2.k, float(swiglu_limit)
        if (self._w13.n != 2 * self.inter or self._w2.n != self.hidden or self.inter % 128
                or self._w13.device != self._w2.device or self._w13.pow2 != self._w2.pow2):
            raise ValueError(f"need w13 [2I, H] and w2 [H, I] with I % 128 == 0, one device and one kind of scales, got "
                             f"{self._w13.n} x {self._w13.k} and {self._w2.n} x {self._w2.k}")

    @classmethod
    def from_float(cls, w13: torch.Tensor, w2: torch.Tensor, *, swiglu_limit: float = 0.0) -> "Fp8SharedExpert":
        """Dense CUDA weights w13 [2I, H] and w2 [H, I] (multiples of 128) -> block-quantised."""
        from .quant import fp8_block_quantize

        return cls(*fp8_block_quantize(w13), *fp8_block_quantize(w2), swiglu_limit=swiglu_limit)

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        a, b = self._w13, self._w2
        rows, ld, out = _rows(x, a, out, b.n)
        m = rows.shape[0]
        if m:
            nbytes = N.lib().asap_fp8_shared_ws_bytes(m, self.hidden, self.inter)
            ws = _scratch(nbytes, a.device)
            with _OnDevice(a.device.index) as stream:
                N.run("asap_fp8_shared", a.handle, b.handle, rows.data_ptr(), ld, m, x.dtype == torch.float16,
                      self.swiglu_limit, out.data_ptr(), ws.data_ptr(), nbytes, a.status, TIMEOUT_NS, stream)
        return out

    def reload(self) -> None:
        """As ``Fp8Linear.reload``, for both weights."""
        self._w13.reload()
        self._w2.reload()

    def release(self) -> None:
        self._w13.release()
        self._w2.release()
