"""Rotary positions of queries and keys in front of the attention, with an optional RMS norm, and their gradient.

    rot = Rotary(128, layout="interleaved", axes=(44, 42, 42))       # frame, row, column of a video latent
    q, k = rot(q, k, positions, q_weight=wq, k_weight=wk)            # q, k [N, H, 128]; positions [3, N]

One kernel turns q and k together (t2t_rotary): every head's pairs by the angle position * frequency, in 32 bits, rounded
once.  Gradients of q, k and the weights pass through it (torch.autograd).  The reference leaves positions to its host.
"""
from __future__ import annotations

import math
import struct

import torch

from torch.autograd.graph import increment_version

from . import _lib
from ._launch import DTYPES, launch
from ._lib import ptr

NORM_NONE, NORM_HEAD, NORM_ROW = 0, 1, 2


def rotary_frequencies(width, base=10000.0, scaling=None):
    """Radians per position of the width / 2 pairs of one axis, and the factor on cosine and sine.

    scaling, for contexts longer than those a model was trained on, is None or a dict with "type" and "factor":

      linear   every frequency divided by the factor
      ntk      the base multiplied by factor^(width / (width - 2)): the fastest pair stays, the slowest is divided by the factor
      yarn     pairs that turn more than `beta_fast` (32) times within `original_length` positions stay, those below `beta_slow`
               (1) turns are divided by the factor, a linear ramp over the pair's number in between; cosine and sine
               multiplied by `attention_factor` (0.1 ln(factor) + 1, and 1 for factors below 1)
      bands    the same by wavelength: below original_length / `high_factor` (4) stay, above original_length / `low_factor` (1)
               divided, in between mixed linearly in the reciprocal of the wavelength
    """
    if width <= 0 or width % 2:
        raise ValueError(f"an axis takes a positive even number of elements, got {width}")
    if not base > 0:
        raise ValueError(f"base must be positive, got {base}")
    s = dict(scaling or {})
    kind, factor = s.pop("type", None), float(s.pop("factor", 1.0))
    if not factor > 0:
        raise ValueError(f"the scaling factor must be positive, got {factor}")
    mscale = 1.0
    if kind == "ntk" and width > 2:
        base = base * factor ** (width / (width - 2))
    freqs = [base ** (-2.0 * j / width) for j in range(width // 2)]
    if kind in (None, "ntk"):
        pass
    elif kind == "linear":
        freqs = [f / factor for f in freqs]
    elif kind in ("yarn", "bands"):
        length = float(s.pop("original_length", 0.0))
        if not length > 0:
            raise ValueError(f"{kind} takes the original_length of the context, got {length}")
        if kind == "yarn" and base == 1:
            raise ValueError("yarn takes a base other than 1: its pairs would all have one wavelength")
        if kind == "yarn":
            fast, slow = float(s.pop("beta_fast", 32.0)), float(s.pop("beta_slow", 1.0))
            pair = lambda turns: width * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
            low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), width - 1)
            kept = [1.0 - min(max((j - low) / max(high - low, 1e-3), 0.0), 1.0) for j in range(width // 2)]
            mscale = float(s.pop("attention_factor", 0.1 * math.log(max(factor, 1.0)) + 1.0))
        else:
            lo, hi = float(s.pop("low_factor", 1.0)), float(s.pop("high_factor", 4.0))
            if not hi > lo:
                raise ValueError("high_factor must be larger than low_factor")
            kept = [min(max((length * f / (2 * math.pi) - lo) / (hi - lo), 0.0), 1.0) for f in freqs]
        freqs = [f * k + f / factor * (1.0 - k) for f, k in zip(freqs, kept)]
    else:
        raise ValueError(f"unknown scaling {kind!r}")
    if s:
        raise ValueError(f"unknown scaling options {sorted(s)} for {kind!r}")
    return freqs, mscale


def _layout(name, t):
    """(batch, token, head) strides of a [N, H, D] or [B, N, H, D] tensor with contiguous heads."""
    st = t.stride()
    if st[-1] != 1 and t.shape[-1] != 1:
        raise ValueError(f"{name}: the elements of a head must be contiguous, got strides {tuple(st)}")
    return (0, st[0], st[1]) if len(st) == 3 else st[:3]


class _Turned(torch.autograd.Function):
    """Rotary.__call__ where autograd wants gradients of its inputs."""

    @staticmethod
    def forward(ctx, rot, q, k, positions, q_weight, k_weight, eps, inverse):
        ctx.rot, ctx.eps, ctx.inverse = rot, eps, inverse
        normed = q_weight is not None
        ctx.save_for_backward(q if normed else None, k if normed else None, positions, q_weight, k_weight)
        return rot(q, k, positions, q_weight=q_weight, k_weight=k_weight, eps=eps, inverse=inverse)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        q, k, positions, q_weight, k_weight = ctx.saved_tensors
        # autograd hands over expanded gradients too
        dq, dk = (d if d is None or d.stride(-1) == 1 else d.contiguous() for d in (dq, dk))
        if q_weight is None:
            return (None, *ctx.rot(dq, dk, positions, inverse=not ctx.inverse), *[None] * 5)
        dq, dk, dwq, dwk = ctx.rot.backward(dq, dk, positions, q=q, k=k, q_weight=q_weight, k_weight=k_weight, eps=ctx.eps)
        return None, dq, dk, None, dwq.to(q_weight.dtype), None if k_weight is None else dwk.to(k_weight.dtype), None, None


_STRIDES4, _STRIDES6 = struct.Struct("12q"), struct.Struct("18q")      # as the C entries take them


class Rotary:
    """Positions of one kind of head.

    head_dim: elements of a head; rotary_dim: how many of them, from the first, are turned (all of them).
    layout: "interleaved" pairs elements (2 j, 2 j + 1), "half" pairs (j, j + rotary_dim / 2).
    axes: widths of the position axes, which add up to rotary_dim; None: one axis.  Axis a's pairs follow those of
        axis a - 1 and have frequencies base^(-2 j / width), j = 0 .. width / 2 - 1.
    scaling: see rotary_frequencies."""

    def __init__(self, head_dim, rotary_dim=None, *, layout="interleaved", base=10000.0, axes=None, scaling=None, device="cuda"):
        rd = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or head_dim % 2 or rd <= 0 or rd % 2 or rd > head_dim or rd > 512:
            raise ValueError(f"head_dim and rotary_dim must be even, rotary_dim at most head_dim and 512; got {head_dim}, {rd}")
        if layout not in ("interleaved", "half"):
            raise ValueError(f"unknown layout {layout!r}")
        widths = (rd,) if axes is None else tuple(axes)
        if sum(widths) != rd:
            raise ValueError(f"axes {widths} do not add up to rotary_dim {rd}")
        self.lib = _lib.load()
        self.head_dim, self.rotary_dim, self.layout, self.axes = head_dim, rd, layout, None if axes is None else widths
        freqs, axis, scales = [], [], set()
        for a, width in enumerate(widths):
            f, m = rotary_frequencies(width, base, scaling)
            freqs += f
            axis += [a] * len(f)
            scales.add(m)
        self.frequencies, self.mscale = freqs, scales.pop()
        # turns per position modulo 1, in units of 2^-64, as the signed 64-bit number of the same bits
        turns = [round(math.fmod(f / (2 * math.pi), 1.0) * 2 ** 64) % 2 ** 64 for f in freqs]
        self.dev = torch.device(device)
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64, device=self.dev)
        self.axis = torch.tensor(axis, dtype=torch.int32, device=self.dev)
        self.dev = self.turns.device
        self._plan = (self.turns.data_ptr(), self.axis.data_ptr())
        self._interleaved = layout == "interleaved"

    # -- checks ------------------------------------------------------------------
    def _check_tensor(self, name, t, like):
        D, shape = self.head_dim, t.shape
        if shape[:-2] == like.shape[:-2] and shape[-1] == D and len(shape) in (3, 4) and t.dtype in DTYPES and t.dtype == like.dtype \
                and t.device == self.dev:
            return
        if t.dim() not in (3, 4) or t.shape[-1] != D or t.dtype not in DTYPES or t.device != self.dev:
            raise ValueError(f"{name}: expected bfloat16, float16 or float32 [N, H, {D}] or [B, N, H, {D}] on {self.dev}, got "
                             f"{t.dtype} {tuple(t.shape)} on {t.device}")
        if t.dim() != like.dim() or t.dtype != like.dtype or t.shape[:-2] != like.shape[:-2]:
            raise ValueError(f"{name}: expected tokens {tuple(like.shape[:-2])} of {like.dtype}, got {t.dtype} {tuple(t.shape)}")

    def _check_positions(self, positions, q):
        want = q.shape[:-2]
        lead = () if self.axes is None else (len(self.axes),)
        B, N = want if len(want) == 2 else (1, want[0])
        shape = positions.shape
        shared = shape == lead + (N,)
        if not shared and shape != lead + (B, N):
            raise ValueError(f"positions: expected {lead + (N,)} or {lead + (B, N)}, got {tuple(shape)}")
        if (positions.dtype != torch.int64 and positions.dtype != torch.int32) or positions.device != self.dev:
            raise ValueError(f"positions: expected int32 or int64 on {self.dev}, got {positions.dtype} on {positions.device}")
        st = positions.stride()
        if st[-1] != 1 and N != 1:
            positions = positions.contiguous()
            st = positions.stride()
        return positions, B, N, st[0] if lead else 0, 0 if shared else st[-2]

    def _check_weights(self, q, k, q_weight, k_weight):
        if q_weight is None and k_weight is None:
            return NORM_NONE, DTYPES[q.dtype]
        if q_weight is None or (k is not None and k_weight is None):
            raise ValueError("q_weight and k_weight are given together")
        D, norm = self.head_dim, None
        for name, t, w in (("q", q, q_weight), ("k", k, k_weight)):
            if t is None:
                continue
            H, size = t.shape[-2], w.numel()
            kind = NORM_HEAD if size == D else NORM_ROW if size == H * D else None
            if kind is None or w.dim() != 1 or not w.is_contiguous() or w.device != self.dev \
                    or w.dtype not in (t.dtype, torch.float32) or w.dtype != q_weight.dtype:
                raise ValueError(f"{name}_weight: expected {t.dtype} or float32 [{D}] (norm of a head) or [{H * D}] (norm of all "
                                 f"heads) on {self.dev}, got {w.dtype} {tuple(w.shape)} on {w.device}")
            if t.shape[-2] == 1 and norm is not None:      # one head: the two norms are the same
                kind = norm
            if norm is not None and kind != norm:
                if name == "k" and q.shape[-2] == 1:
                    norm = kind
                else:
                    raise ValueError("q_weight and k_weight ask for different norms")
            norm = kind
        return norm, DTYPES[q_weight.dtype]

    def _outputs(self, q, k, out):
        if out is None:
            new, dense = torch.empty_like, torch.contiguous_format
            return new(q, memory_format=dense), None if k is None else new(k, memory_format=dense)
        qo, ko = out
        for name, o, t in (("q", qo, q), ("k", ko, k)):
            if (o is None) != (t is None) or (o is not None and (o.shape != t.shape or o.dtype != t.dtype or o.device != t.device)):
                raise ValueError(f"out: expected a tensor like {name}")
        return qo, ko

    def _common(self, q, k, positions):
        self._check_tensor("q", q, q)
        if k is not None:
            self._check_tensor("k", k, q)
        return self._check_positions(positions, q)

    # -- calls -------------------------------------------------------------------
    def __call__(self, q, k, positions, *, q_weight=None, k_weight=None, eps=1e-6, out=None, inverse=False):
        """q [N, H, D] or [B, N, H, D] and k (the same with its own number of heads, or None), positions int32 or int64
        [N] or [B, N], with axes [A, N] or [A, B, N].  Any strides with contiguous heads.  q_weight, k_weight [D] or
        [H * D]: RMS norm over each head or over all heads of a token in front of the rotation.  inverse: turns back,
        which without a norm is the gradient.  out: (q, k) to write to, which may be the inputs and share no other memory with
        them; not where autograd wants a gradient.  Returns (q, k)."""
        checked, B, N, pa, pb = self._common(q, k, positions)
        norm, wd = self._check_weights(q, k, q_weight, k_weight)
        if norm and inverse:
            raise ValueError("inverse takes no norm: see backward")
        if (q.requires_grad or k is not None and k.requires_grad or q_weight is not None
                and (q_weight.requires_grad or k_weight is not None and k_weight.requires_grad)
                or out is not None and any(t is not None and t.requires_grad for t in out)) and torch.is_grad_enabled():
            if out is not None:
                raise ValueError("out: an input or output requires a gradient")
            return _Turned.apply(self, q, k, positions, q_weight, k_weight, eps, inverse)
        positions = checked
        qo, ko = self._outputs(q, k, out)
        if out is not None:
            increment_version([t for t in out if t is not None])
        if B * N == 0:
            return qo, ko
        if q.shape[-2] == 0:      # k alone
            if k is not None:
                self(k, None, positions, q_weight=k_weight, eps=eps, out=(ko, None), inverse=inverse)
            return qo, ko
        Hk = 0 if k is None else k.shape[-2]
        kk, kko = (k, ko) if Hk else (q, qo)
        strides = _STRIDES4.pack(*_layout("q", q), *_layout("k", kk), *_layout("out", qo), *_layout("out", kko))
        launch(self.dev, "t2t_rotary", self.lib.t2t_rotary, q.data_ptr(), ptr(k), qo.data_ptr(), ptr(ko), ptr(q_weight), ptr(k_weight),
               wd, positions.data_ptr(), 8 if positions.dtype == torch.int64 else 4, pa, pb, *self._plan, strides, B, N, q.shape[-2],
               Hk, self.head_dim, self.rotary_dim, self._interleaved, bool(inverse), norm, self.mscale, eps, DTYPES[q.dtype])
        return qo, ko

    def backward(self, dq, dk, positions, *, q=None, k=None, q_weight=None, k_weight=None, eps=1e-6, out=None):
        """Gradients of the inputs from those of the outputs: (dq, dk, dq_weight, dk_weight), the last two in fp32 and None
        without a norm.  With a norm q and k are the inputs of the call.  out: (dq, dk) to write to, which may be the
        gradients that are read.  What autograd runs; for those who keep their own inputs."""
        if q_weight is None and k_weight is None:
            return (*self(dq, dk, positions, out=out, inverse=True), None, None)
        positions, B, N, pa, pb = self._common(dq, dk, positions)
        if q is None or (dk is not None and k is None):
            raise ValueError("the gradient of the norm needs q and k")
        k = None if dk is None else k
        for name, t, d in (("q", q, dq), ("k", k, dk)):
            if t is not None:
                self._check_tensor(name, t, d)
                if t.shape != d.shape:
                    raise ValueError(f"{name}: expected {tuple(d.shape)}, got {tuple(t.shape)}")
        norm, wd = self._check_weights(q, k, q_weight, k_weight)
        qo, ko = self._outputs(dq, dk, out)
        if out is not None:
            increment_version([t for t in out if t is not None])
        dwq = torch.empty(q_weight.shape[0], dtype=torch.float32, device=self.dev)
        dwk = None if k is None else torch.empty(k_weight.shape[0], dtype=torch.float32, device=self.dev)
        H, Hk, D = q.shape[-2], 0 if k is None else k.shape[-2], self.head_dim
        if H == 0 and Hk and B * N:
            ko, _, dwk, _ = self.backward(dk, None, positions, q=k, q_weight=k_weight, eps=eps, out=(ko, None))
            return qo, ko, dwq.zero_(), dwk
        if B * N == 0 or H == 0:
            return qo, ko, dwq.zero_(), None if dwk is None else dwk.zero_()
        side_k = (k, dk, ko) if Hk else (q, dq, qo)
        strides = _STRIDES6.pack(*_layout("q", q), *_layout("k", side_k[0]), *_layout("dq", dq), *_layout("dk", side_k[1]),
                                 *_layout("out", qo), *_layout("out", side_k[2]))
        ws = torch.empty(int(self.lib.t2t_rotary_grad_ws_bytes(H, Hk, D, norm)), dtype=torch.uint8, device=self.dev)
        launch(self.dev, "t2t_rotary_grad", self.lib.t2t_rotary_grad, ptr(dq), ptr(dk), ptr(q), ptr(k), ptr(qo), ptr(ko),
               ptr(q_weight), ptr(k_weight), wd, ptr(dwq), ptr(dwk), ptr(positions), positions.element_size(), pa, pb, *self._plan,
               strides, B, N, H, Hk, D, self.rotary_dim, self._interleaved, norm, self.mscale, eps, DTYPES[q.dtype], ptr(ws),
               ws.numel())
        return qo, ko, dwq, dwk


def latent_positions(frames, rows, columns, *, start=0, count=None, device="cuda"):
    """[3, n] int64 positions (frame, row, column) of the row-major tokens of a video latent, or of `count` of them from
    token `start` (one rank's share)."""
    total = frames * rows * columns
    n = torch.arange(start, total if count is None else start + count, device=device)
    return torch.stack((n // (rows * columns), n // columns % rows, n % columns))
