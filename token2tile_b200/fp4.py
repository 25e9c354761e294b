"""Microscaled 4-bit floating point around the attention: quantisation, products, and the linear layers made of them.

    w = Fp4Linear(weight, bias)                                  # weight [out, in] bf16, quantised once
    y = w(x, shift=shift, scale=scale)                           # modulated layer norm, quantisation, product
    x = Fp4FeedForward(up, down)(x, shift=..., scale=..., gate=..., residual=x)

Formats: "mxfp4" (blocks of 32, scale a power of two) and "nvfp4" (blocks of 16, scale an 8-bit float with 3 mantissa bits, and
one scale for the whole matrix).  Elements are 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.  The products run on the
4-bit tensor cores and sum in 32 bits.  No gradients pass through any of these: their results require none.
"""
from __future__ import annotations

import ctypes
import math
import threading

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._launch import DTYPES, launch
from ._lib import ptr

FORMATS = {"mxfp4": 0, "nvfp4": 1}
BLOCK = {"mxfp4": 32, "nvfp4": 16}
ACTIVATIONS = {None: 0, "gelu_tanh": 1, "silu": 2}
FEW_ROWS = 4      # T2T_FP4_FEW_ROWS
WIDE_VECTORS = 0x100      # T2T_WIDE_VECTORS


class _Status:
    """One word of pinned host memory per device that a kernel whose bounded wait gave up writes to."""

    def __init__(self):
        self.word = torch.zeros(1, dtype=torch.int32).pin_memory()
        self.ptr = self.word.data_ptr()
        self.value = ctypes.c_int.from_address(self.ptr)


_status: dict = {}
_status_lock = threading.Lock()      # queued kernels point to the word: a device has one, whichever thread asks first


def _status_of(dev):
    s = _status.get(dev.index)
    if s is None:
        if dev.index is None:
            raise ValueError(f"expected tensors on a CUDA device, got {dev}")
        with _status_lock:
            s = _status.get(dev.index)
            if s is None:
                s = _status[dev.index] = _Status()
    return s


def check_status(device="cuda", *, wait=True):
    """Raises RuntimeError if a product on this device gave up a wait; `wait` waits for the device's work first.  Every product
    looks at the word of the earlier ones before it is queued."""
    dev = torch.device(device)
    dev = torch.device("cuda", torch.cuda.current_device()) if dev.index is None else dev
    if wait:
        torch.cuda.synchronize(dev)
    s = _status_of(dev)
    if s.value.value:
        code, s.value.value = s.value.value, 0
        raise RuntimeError(f"fp4_matmul: {_lib.STATUS.get(code, code)}")


def _fmt(fmt):
    if fmt not in FORMATS:
        raise ValueError(f"unknown format {fmt!r}: expected one of {sorted(FORMATS)}")
    return FORMATS[fmt]


class Fp4Tensor:
    """A quantised matrix [rows, K] on a GPU: `codes` and `scales` (views of one buffer, `data`; their layouts: t2t_fp4_quantize in
    the C header), `fmt` and `tensor_scale`."""

    __slots__ = ("data", "shape", "fmt", "tensor_scale", "device", "_split")

    def __init__(self, data, shape, fmt, tensor_scale=1.0):
        self.data, self.shape, self.fmt, self.tensor_scale = data, shape, fmt, tensor_scale
        self.device = data.device
        self._split = shape[0] * (-(-shape[1] // 32) * 16)      # bytes of the codes

    @property
    def codes(self):
        return self.data[:self._split].view(self.shape[0], -1 if self.shape[0] else -(-self.shape[1] // 32) * 16)

    @property
    def scales(self):
        return self.data[self._split:]

    def pointers(self):
        at = self.data.data_ptr()
        return at, at + self._split

    def __repr__(self):
        return f"Fp4Tensor({list(self.shape)}, {self.fmt}, tensor_scale={self.tensor_scale}, {self.device})"

    @staticmethod
    def empty(rows, K, fmt, tensor_scale=1.0, device="cuda"):
        _fmt(fmt)
        if rows < 0 or K <= 0:
            raise ValueError(f"expected rows >= 0 and K > 0, got {rows}, {K}")
        if not 2.0 ** -100 <= tensor_scale <= 2.0 ** 100:
            raise ValueError(f"tensor_scale: expected 2^-100 .. 2^100, got {tensor_scale}")
        size = rows * (-(-K // 32) * 16) + -(-rows // 128) * -(-K // (4 * BLOCK[fmt])) * 512
        return Fp4Tensor(torch.empty(size, dtype=torch.uint8, device=device), (rows, K), fmt, float(tensor_scale))

    @staticmethod
    def from_stored(packed, scales, K, fmt, *, tensor_scale=1.0):
        """A matrix as checkpoints hold it: packed uint8 [rows, ceil(K / 2)], the even element in the lower four bits, and
        scales [rows, ceil(K / block)], uint8 or the 8-bit float type of the format."""
        _fmt(fmt)
        rows, blocks = packed.shape[0], -(-K // BLOCK[fmt])
        if scales.dtype in (torch.float8_e4m3fn, torch.float8_e8m0fnu):
            if (scales.dtype == torch.float8_e4m3fn) != (fmt == "nvfp4"):
                raise ValueError(f"scales: {scales.dtype} is not the type of {fmt}")
            scales = scales.view(torch.uint8)
        if packed.dtype != torch.uint8 or tuple(packed.shape) != (rows, -(-K // 2)) or scales.dtype != torch.uint8 \
                or tuple(scales.shape) != (rows, blocks) or scales.device != packed.device or not packed.is_cuda:
            raise ValueError(f"expected CUDA uint8 [rows, {-(-K // 2)}] and [rows, {blocks}], got {packed.dtype} "
                             f"{tuple(packed.shape)} and {scales.dtype} {tuple(scales.shape)} on {packed.device}, {scales.device}")
        t = Fp4Tensor.empty(rows, K, fmt, tensor_scale, packed.device)
        t.codes.zero_()[:, :packed.shape[1]] = packed
        if K % 2:
            t.codes[:, K // 2] &= 15
        slabs, atoms = -(-rows // 128), -(-blocks // 4)
        s = torch.zeros(slabs * 128, atoms * 4, dtype=torch.uint8, device=packed.device)
        s[:rows, :blocks] = scales
        # row = 128 slab + 32 word + lane, block = 4 atom + byte  ->  [slab, atom, lane, word, byte]
        t.scales.copy_(s.view(slabs, 4, 32, atoms, 4).permute(0, 3, 2, 1, 4).reshape(-1))
        return t

    def to_stored(self):
        """(packed, scales), the inverse of from_stored."""
        (rows, K), blocks = self.shape, -(-self.shape[1] // BLOCK[self.fmt])
        slabs, atoms = -(-rows // 128), -(-blocks // 4)
        s = self.scales.view(slabs, atoms, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(slabs * 128, atoms * 4)
        return self.codes[:, :-(-K // 2)].contiguous(), s[:rows, :blocks].contiguous()

    def dequantize(self, dtype=torch.float32, out=None):
        """The values, [rows, K]."""
        rows, K = self.shape
        if out is None:
            if dtype not in DTYPES:
                raise ValueError(f"dtype: expected bfloat16, float16 or float32, got {dtype}")
            out = torch.empty(rows, K, dtype=dtype, device=self.device)
        elif tuple(out.shape) != self.shape or out.dtype not in DTYPES or out.device != self.device \
                or (out.stride(1) != 1 and K != 1):
            raise ValueError(f"out: expected [{rows}, {K}] with contiguous rows on {self.device}")
        else:
            increment_version(out)
        if rows:
            launch(self.device, "t2t_fp4_dequantize", _lib.load().t2t_fp4_dequantize, *self.pointers(), rows, K, FORMATS[self.fmt],
                   self.tensor_scale, out.data_ptr(), out.stride(0) if rows > 1 else K, DTYPES[out.dtype])
        return out


def _rows(name, x):
    """x [..., K] as a [rows, K] view with contiguous rows."""
    if x.dtype not in DTYPES or not x.is_cuda or x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"{name}: expected a CUDA bfloat16, float16 or float32 tensor [..., K], got {x.dtype} "
                         f"{tuple(x.shape)} on {x.device}")
    if x.dim() != 2:
        try:
            x = x.view(-1, x.shape[-1]) if x.numel() else x.new_empty(0, x.shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}: rows must be evenly spaced, got strides {tuple(x.stride())}") from None
    if x.stride(1) != 1 and x.shape[1] != 1:
        raise ValueError(f"{name}: the elements of a row must be contiguous, got strides {tuple(x.stride())}")
    return x


def _vector(name, v, n, dev, dtype=None):
    if v is not None and (v.dim() != 1 or v.shape[0] != n or not v.is_contiguous() or v.device != dev or v.dtype not in DTYPES
                          or (dtype is not None and v.dtype != dtype)):
        raise ValueError(f"{name}: expected a contiguous {dtype or 'floating'} [{n}] on {dev}, got {v.dtype} {tuple(v.shape)} "
                         f"on {v.device}")


def _modulation(shift, scale, K, dev, dtype):
    """Checks of shift and scale, of which there is one; the C entries' type of an x of `dtype` with them."""
    if shift is None or scale is None:
        raise ValueError("shift and scale are given together")
    kind = torch.float32 if shift.dtype == torch.float32 else dtype
    _vector("shift", shift, K, dev, kind)
    _vector("scale", scale, K, dev, kind)
    return DTYPES[dtype] if kind == dtype else DTYPES[dtype] | WIDE_VECTORS


def _vector_type(bias, gate):
    vec = bias if bias is not None else gate
    return 0 if vec is None else DTYPES[vec.dtype]


def _shares(p, size, q, other):
    """Two ranges of bytes have some in common."""
    return p < q + other and q < p + size


def _beside(residual, out):
    """The residual rows, or a copy where some of their elements are other elements of out [M, N]: those would be overwritten before
    they are read."""
    (M, N), size, p, q = out.shape, out.element_size(), residual.data_ptr(), out.data_ptr()
    rs, os = residual.stride(0) if M > 1 else N, out.stride(0) if M > 1 else N
    if (p == q and rs == os) or not _shares(p, ((M - 1) * rs + N) * size, q, ((M - 1) * os + N) * size):
        return residual
    if rs == os:      # columns of one wide matrix: `down` rows and `right` elements further on, or one row more and to the left
        down, right = divmod(q - p, rs * size)
        if not (right < N * size and abs(down) < M) and not ((rs * size - right) < N * size and abs(down + 1) < M):
            return residual
    return residual.clone()


def fp4_quantize(x, fmt="nvfp4", *, tensor_scale=1.0, shift=None, scale=None, eps=1e-6, out=None):
    """x [..., K] as an Fp4Tensor of its rows.  A block's scale comes from its largest magnitude: 2^(floor(log2 top) - 2)
    ("mxfp4") or the 8-bit float next to top / 6 / tensor_scale ("nvfp4"); its elements go to the nearest code, ties to the
    even one, saturating at 6.  A block with a NaN or an infinity is NaN as a whole.

    shift, scale [K] of x's type or float32: quantises layer_norm(x) * (1 + scale) + shift, which is never written out.  (A norm's
    weight w as scale = w - 1 is given in float32: in 16 bits the difference loses what w has below 2^-8.)"""
    x = _rows("x", x)
    M, K = x.shape
    kind = DTYPES[x.dtype] if shift is None and scale is None else _modulation(shift, scale, K, x.device, x.dtype)
    given = out is not None
    if not given:
        out = Fp4Tensor.empty(M, K, fmt, tensor_scale, x.device)
    elif out.shape != (M, K) or out.fmt != fmt or out.device != x.device:
        raise ValueError(f"out: expected [{M}, {K}] {fmt} on {x.device}, got {out}")
    if not 2.0 ** -100 <= tensor_scale <= 2.0 ** 100 or (fmt == "mxfp4" and tensor_scale != 1):
        raise ValueError(f"tensor_scale: expected 1 (mxfp4) or 2^-100 .. 2^100 (nvfp4), got {tensor_scale}")
    out.tensor_scale = float(tensor_scale)
    if given:
        increment_version(out.data)
    if M:
        launch(x.device, "t2t_fp4_quantize", _lib.load().t2t_fp4_quantize, x.data_ptr(), x.stride(0), ptr(shift), ptr(scale), eps, M,
               K, kind, _fmt(fmt), tensor_scale, *out.pointers())
    return out


def fp4_matmul(a, w, *, bias=None, activation=None, gate=None, residual=None, dtype=torch.bfloat16, out=None):
    """residual + gate * activation(a w^T + bias) for Fp4Tensors a [M, K] and w [N, K] of one format: [M, N] of `dtype`, summed
    in 32 bits and rounded once.  bias, gate [N] of one type; activation None, "gelu_tanh" or "silu"; residual [M, N] of the
    result's type; out may be the residual, and shares no memory with the other inputs.

    dtype "mxfp4" or "nvfp4" (the format of a and w), or an Fp4Tensor [M, N] as out: the result quantised as by fp4_quantize,
    from 32 bits; takes no residual.

    The tensor scales' product is a factor in 32 bits: one of 2^128 or more is refused, one below 2^-149 is 0."""
    (M, K), (N, Kw) = a.shape, w.shape
    dev = a.device
    if K != Kw or a.fmt != w.fmt or w.device != dev:
        raise ValueError(f"expected matrices of one format, width and device, got {a} and {w}")
    alpha = a.tensor_scale * w.tensor_scale
    if alpha >= 2.0 ** 128:
        raise ValueError(f"tensor scales {a.tensor_scale} and {w.tensor_scale}: their product leaves the range of 32 bits")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    _vector("bias", bias, N, dev)
    _vector("gate", gate, N, dev, None if bias is None else bias.dtype)
    given = out is not None
    codes = isinstance(out, Fp4Tensor) or (out is None and dtype in FORMATS)
    if codes:
        if residual is not None or (dtype if out is None else out.fmt) != a.fmt:
            raise ValueError(f"a quantised result has the format of its factors, {a.fmt}, and no residual")
        if out is None:
            out = Fp4Tensor.empty(M, N, a.fmt, 1.0, dev)
        elif any(_shares(t.data.data_ptr(), t.data.numel(), out.data.data_ptr(), out.data.numel()) for t in (a, w)):
            raise ValueError("out: shares memory with a factor")
    elif out is None:
        if dtype not in DTYPES:
            raise ValueError(f"dtype: expected bfloat16, float16, float32 or {a.fmt!r}, got {dtype}")
        out = torch.empty(M, N, dtype=dtype, device=dev)
    for name, t in (("out", out), ("residual", residual)):
        if t is not None and (tuple(t.shape) != (M, N) or t.device != dev or not codes and (
                t.dtype != out.dtype or t.dtype not in DTYPES or (t.stride(1) != 1 and N != 1))):
            raise ValueError(f"{name}: expected [{M}, {N}] of the result's type with contiguous rows on {dev}, got {t!r}"[:300])
    if given:
        increment_version(out.data if codes else out)
    if M == 0 or N == 0:
        return out
    if residual is not None:
        residual = _beside(residual, out)
    status = _status_of(dev)
    if status.value.value:
        check_status(dev, wait=False)
    head = (*a.pointers(), *w.pointers(), M, N, K, FORMATS[a.fmt], alpha, ptr(bias),
            ACTIVATIONS[activation], ptr(gate), _vector_type(bias, gate))
    if codes:
        launch(dev, "t2t_fp4_matmul_quantize", _lib.load().t2t_fp4_matmul_quantize, *head, out.tensor_scale, *out.pointers(),
               status.ptr)
    else:
        launch(dev, "t2t_fp4_matmul", _lib.load().t2t_fp4_matmul, *head, ptr(residual), 0 if residual is None else residual.stride(0),
               out.data_ptr(), out.stride(0) if M > 1 else N, DTYPES[out.dtype], status.ptr)
    return out


def fp4_tensor_scale(x):
    """The smallest power of two that keeps every block scale of x within the range of "nvfp4" (reads x's largest magnitude
    back: for weights, once)."""
    top = float(x.abs().amax()) if x.numel() else 0.0
    if not math.isfinite(top):
        raise ValueError("fp4_tensor_scale: non-finite input")
    return min(max(2.0 ** math.ceil(math.log2(max(top, 1e-30) / (6 * 448))), 2.0 ** -100), 2.0 ** 100)


class Fp4Linear:
    """y = activation(x W^T + b) with W [out, in] quantised once and every x on the way in; plain tensors, no autograd.

    x is quantised with a tensor scale of 1: "nvfp4" holds blocks whose largest magnitude is between 0.006 and 2,688 (below 0.1 with
    fewer bits of scale), saturates above and gives zeros below.  Rows beyond that are quantised by fp4_quantize with a tensor_scale
    of their own and given so."""

    def __init__(self, weight, bias=None, *, fmt="nvfp4"):
        if isinstance(weight, Fp4Tensor):
            self.w = weight
        else:
            if weight.dim() != 2:
                raise ValueError(f"weight: expected [out, in], got {tuple(weight.shape)}")
            self.w = fp4_quantize(weight, fmt, tensor_scale=fp4_tensor_scale(weight) if fmt == "nvfp4" else 1.0)
        _vector("bias", bias, self.w.shape[0], self.w.device)
        self.b = bias

    def __call__(self, x, *, shift=None, scale=None, eps=1e-6, activation=None, gate=None, residual=None, out=None, dtype=None):
        """x [..., in] -> [..., out] of x's type.  shift, scale [in] of that type or float32: of layer_norm(x) * (1 + scale) + shift.
        gate [out], residual and out [..., out]: residual + gate * (...).  x may be an Fp4Tensor [rows, in] that several layers
        share (fp4_quantize); the result is then of `dtype` (bfloat16)."""
        if isinstance(x, Fp4Tensor):
            if shift is not None or scale is not None:
                raise ValueError("shift and scale go into the quantisation of x")
            return fp4_matmul(x, self.w, bias=self.b, activation=activation, gate=gate, residual=residual,
                              dtype=dtype or torch.bfloat16, out=out)
        if dtype is not None and dtype != x.dtype:
            raise ValueError(f"dtype: the result has the type of x, {x.dtype}")
        K = self.w.shape[1]
        if x.shape[-1] != K:
            raise ValueError(f"x: expected [..., {K}], got {tuple(x.shape)}")
        w = self.w
        inside = out is None and shift is None and math.prod(x.shape[:-1]) <= FEW_ROWS      # quantised by the product
        rows, kind, M, y, to, res, ws = _layer(x, K, w, self.b, shift, scale, gate, residual, out, activation,
                                               0 if inside else _bytes(x.shape, K, w.fmt))
        if M:
            dev = w.device
            launch(dev, "t2t_fp4_linear", _lib.load().t2t_fp4_linear, rows.data_ptr(), rows.stride(0), ptr(shift), ptr(scale), eps, M,
                   K, kind, FORMATS[w.fmt], *w.pointers(), w.tensor_scale, w.shape[0], ptr(self.b),
                   ACTIVATIONS[activation], ptr(gate), _vector_type(self.b, gate), ptr(res), 0 if res is None else res.stride(0),
                   to.data_ptr(), to.stride(0) if M > 1 else w.shape[0], ptr(ws), 0 if ws is None else ws.shape[0], _status_of(dev).ptr)
        return y


def _bytes(shape, K, fmt):
    """Bytes of a quantised matrix of the rows of a tensor of this shape, K wide."""
    M = math.prod(shape[:-1])
    return M * (-(-K // 32) * 16) + -(-M // 128) * -(-K // (4 * BLOCK[fmt])) * 512


def _layer(x, K, last, bias, shift, scale, gate, residual, out, activation, ws_bytes):
    """Checks of a layer whose last product is with `last`, and what it needs: x as rows, its type with the vectors', the rows' number (0:
    nothing to do), the result, it and the residual as rows, workspace."""
    dev, shape = last.device, (*x.shape[:-1], last.shape[0])
    N = shape[-1]
    if x.device != dev:
        raise ValueError(f"x: expected a tensor on {dev}, got {x.device}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    rows = _rows("x", x)
    kind = DTYPES[x.dtype] if shift is None and scale is None else _modulation(shift, scale, K, dev, x.dtype)
    _vector("gate", gate, N, dev, None if bias is None else bias.dtype)
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (t.shape != shape or t.dtype != x.dtype or t.device != dev):
            raise ValueError(f"{name}: expected {x.dtype} {shape} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if out is None:
        y = torch.empty(*shape, dtype=x.dtype, device=dev)
    else:
        y = out
        increment_version(y)
    M = rows.shape[0]
    if M == 0 or N == 0:
        return rows, kind, 0, y, None, None, None
    if _status_of(dev).value.value:
        check_status(dev, wait=False)
    to = _rows("out", y)
    if residual is not None:
        residual = _rows("residual", residual) if out is None else _beside(_rows("residual", residual), to)
    return (rows, kind, M, y, to, residual,
            torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None)


class Fp4FeedForward:
    """residual + gate * down(activation(up(layer_norm(x) * (1 + scale) + shift))).  What lies between the two products is
    quantised from 32 bits, without a rounding to 16 in between, and with a tensor scale of 1 as x is (Fp4Linear); hidden values beyond
    its range go through fp4_matmul into an Fp4Tensor with a scale of their own."""

    def __init__(self, up, down, activation="gelu_tanh"):
        if up.w.shape[0] != down.w.shape[1] or up.w.fmt != down.w.fmt or up.w.device != down.w.device:
            raise ValueError(f"up {up.w} and down {down.w} do not follow each other")
        if activation not in ACTIVATIONS:
            raise ValueError(f"unknown activation {activation!r}")
        self.up, self.down, self.activation = up, down, activation

    def __call__(self, x, *, shift=None, scale=None, eps=1e-6, gate=None, residual=None, out=None):
        K = self.up.w.shape[1]
        if x.shape[-1] != K:
            raise ValueError(f"x: expected [..., {K}], got {tuple(x.shape)}")
        up, down = self.up, self.down
        u, d = up.w, down.w
        F, N = d.shape[1], d.shape[0]
        rows, kind, M, y, to, res, ws = _layer(x, K, d, down.b, shift, scale, gate, residual, out, self.activation,
                                               _bytes(x.shape, K, u.fmt) + _bytes(x.shape, F, u.fmt))
        if M:
            dev = u.device
            launch(dev, "t2t_fp4_feed_forward", _lib.load().t2t_fp4_feed_forward, rows.data_ptr(), rows.stride(0), ptr(shift),
                   ptr(scale), eps, M, K, kind, FORMATS[u.fmt], *u.pointers(), u.tensor_scale, F, ptr(up.b),
                   _vector_type(up.b, None), ACTIVATIONS[self.activation], *d.pointers(), d.tensor_scale, N, ptr(down.b), ptr(gate),
                   _vector_type(down.b, gate), ptr(res), 0 if res is None else res.stride(0), to.data_ptr(),
                   to.stride(0) if M > 1 else N, ws.data_ptr(), ws.shape[0], _status_of(dev).ptr)
        return y
