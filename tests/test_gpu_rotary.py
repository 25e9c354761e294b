"""Rotary positions with their norm and gradient against the definition in 64 bits.

Tolerances.  Outputs are rounded once: half a unit in the last place, 2^-9 (bfloat16), 2^-12 (half) or 2^-25 (float) of the
result, doubled for results at a power of two.  Behind that everything is in 32 bits: the angle (2^-25 half turns, 1e-7
rad), sine and cosine (1.2e-7), the sums of squares (threads add up to some hundred terms one after the other: 1e-5, halved by
the square root, in the worst case; 1e-6 is typical) and a few products: 4e-6 of the row's largest result."""
import ctypes
import math

import pytest
import torch

import plain64
from token2tile_b200 import Rotary, latent_positions

pytestmark = pytest.mark.gpu
DEV = "cuda"
ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def close(got, want, dtype, dims=(-2, -1)):
    err = (got.double().cpu() - want).abs()
    tol = ULP[dtype] * want.abs() + 4e-6 * want.abs().amax(dims, keepdim=True) + 1e-30 + (2.0 ** -25 if dtype == F16 else 0)
    assert bool((err <= tol).all()), float((err / tol).max())


def make(shape, dtype, gen, packed=False, kv=0):
    """Two tensors [.., N, H or kv, D]; packed: views of one tensor with another head behind them."""
    *lead, H, D = shape
    if packed:
        t = torch.randn(*lead, H + kv + 1, D, generator=gen).to(dtype).to(DEV)
        return t[..., :H, :], t[..., H:H + kv, :]
    return torch.randn(*lead, H, D, generator=gen).to(dtype).to(DEV), torch.randn(*lead, kv, D, generator=gen).to(dtype).to(DEV)


def axis_of(rot):
    return rot.axis.cpu().tolist()


CASES = [
    # N, H, Hk, D, rd, layout, axes, norm, dtype, packed, start
    (1, 40, 8, 128, 128, "half", None, "", BF, True, 1000003),
    (3, 2, 2, 128, 128, "interleaved", (44, 42, 42), "row", BF, False, 0),
    (37, 40, 40, 128, 128, "interleaved", (44, 42, 42), "row", BF, False, 0),
    (5, 12, 12, 128, 128, "interleaved", None, "head", F16, False, 7),
    (33, 3, 1, 64, 32, "half", None, "head", F32, True, 131000),
    (9, 5, 5, 80, 40, "half", None, "row", BF, True, 0),
    (9, 5, 2, 96, 48, "interleaved", (16, 16, 16), "head", F16, False, 0),
    (4, 1, 1, 256, 256, "half", None, "row", F32, False, 12),
    (4, 3, 1, 6, 2, "interleaved", None, "row", BF, False, 12),
    (4, 3, 1, 10, 6, "half", None, "head", F32, True, 12),
    (2, 40, 40, 512, 512, "half", None, "row", BF, False, 3),
    (2, 7, 7, 1024, 512, "interleaved", None, "head", BF, False, 3),
    # enough tokens that blocks take several each, with one, two and four items a thread
    (700, 3, 3, 64, 32, "interleaved", None, "head", F32, False, 9),
    (410, 12, 12, 128, 128, "interleaved", (44, 42, 42), "row", BF, False, 0),
    (1300, 12, 4, 128, 128, "half", None, "head", BF, True, 0),
    (900, 32, 8, 128, 64, "half", None, "head", F16, True, 0),
    (620, 40, 40, 128, 128, "interleaved", (44, 42, 42), "row", BF, False, 0),
    (160, 40, 40, 128, 128, "half", None, "row", F32, False, 5),
    (450, 5, 1, 256, 256, "half", None, "row", F16, False, 5),
    (300, 64, 64, 128, 64, "interleaved", None, "", BF, False, 5),
    (200, 100, 3, 128, 128, "half", None, "head", BF, False, 5),
    (1000, 1, 1, 8, 8, "interleaved", None, "row", F16, False, 5),
    (333, 7, 2, 80, 40, "half", None, "row", BF, True, 0),
]


@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize("batch", [0, 2])
def test_forward_and_gradient(case, batch):
    N, H, Hk, D, rd, layout, axes, norm, dtype, packed, start = case
    gen = torch.Generator().manual_seed(N * 1000 + D)
    rot = Rotary(D, rd, layout=layout, axes=axes, base=10000.0, device=DEV)
    lead = (batch, N) if batch else (N,)
    q, k = make((*lead, H, D), dtype, gen, packed, Hk)
    dq, dk = make((*lead, H, D), dtype, gen, packed, Hk)
    A = 1 if axes is None else len(axes)
    pos = torch.randint(0, 1000, (A, *lead), generator=gen) + start
    positions = (pos if axes else pos[0]).to(DEV)
    qw = kw = None
    if norm:
        qw, kw = ((1 + 0.2 * torch.randn(h * D if norm == "row" else D, generator=gen)).to(dtype).to(DEV) for h in (H, Hk))
    before = [t.clone() for t in (q, k)]
    got = rot(q, k, positions, q_weight=qw, k_weight=kw)
    back = rot.backward(dq, dk, positions, q=q, k=k, q_weight=qw, k_weight=kw)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    args = (pos, rot.frequencies, axis_of(rot))
    for i, (x, dy, w) in enumerate(((q, dq, qw), (k, dk, kw))):
        w = None if w is None else w.cpu()
        x, dy = x.double().cpu(), dy.double().cpu()
        close(got[i], plain64.rotary(x, w, 1e-6, *args, layout=layout), dtype)
        dx, dw = plain64.rotary_grad(dy, x, w, 1e-6, *args, layout=layout)
        close(back[i], dx, dtype)
        if w is None:
            assert back[2] is None and back[3] is None
        else:
            assert back[2 + i].dtype == F32
            # sums over the tokens (and heads) in 32 bits on top of the above
            g = plain64.rotate(dy, *args, layout=layout, inverse=True)
            size = (g * plain64.rms(x, torch.ones_like(w), 1e-6)).abs()
            size = (size.flatten(-2) if norm == "row" and H * D != D else size).reshape(-1, w.numel()).sum(0)
            err = (back[2 + i].double().cpu() - dw).abs()
            assert bool((err <= 1e-5 * size + 1e-6).all()), float(err.max())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_in_place_and_out(dtype):
    gen = torch.Generator().manual_seed(4)
    rot = Rotary(128, axes=(44, 42, 42))
    q, k = make((50, 12, 128), dtype, gen, False, 12)
    pos = latent_positions(2, 5, 5)
    w = torch.rand(12 * 128, generator=gen).to(DEV)      # 32-bit weights with tensors of 16 bits
    want = rot(q, k, pos, q_weight=w, k_weight=w)
    dq, dk = make((50, 12, 128), dtype, gen, False, 12)
    grads = rot.backward(dq, dk, pos, q=q, k=k, q_weight=w, k_weight=w)
    again = rot.backward(dq, dk, pos, q=q, k=k, q_weight=w, k_weight=w, out=(dq, dk))
    assert again[0] is dq and all(torch.equal(a, b) for a, b in zip(grads, again))
    # head-major outputs, as the attention reads them
    out = tuple(torch.empty(12, 50, 128, dtype=dtype, device=DEV).transpose(0, 1) for _ in range(2))
    rot(q, k, pos, q_weight=w, k_weight=w, out=out)
    assert all(torch.equal(a, b) for a, b in zip(want, out))
    rot(q, k, pos.to(torch.int32), q_weight=w, k_weight=w, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_same_bits_every_time_and_on_another_stream():
    gen = torch.Generator().manual_seed(5)
    rot = Rotary(128)
    q, k = make((777, 12, 128), BF, gen, False, 12)
    w = torch.rand(12 * 128, generator=gen).to(BF).to(DEV)
    pos = torch.arange(777, device=DEV)
    want = rot.backward(q, k, pos, q=q, k=k, q_weight=w, k_weight=w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = rot.backward(q, k, pos, q=q, k=k, q_weight=w, k_weight=w)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_gradient_of_the_kernels_against_differences():
    """Directional derivative of the forward kernel in 32 bits: differences over 2 h = 0.04 are off by h^2 (third derivatives of
    order one) and by rounding, 1e-6 / h."""
    gen = torch.Generator().manual_seed(6)
    rot = Rotary(16, 8, layout="half")
    q, k = make((6, 3, 16), F32, gen, False, 3)
    w = (1 + 0.1 * torch.randn(48, generator=gen)).to(DEV)
    pos = torch.arange(6, device=DEV) * 50
    dq, dk = make((6, 3, 16), F32, gen, False, 3)
    got = rot.backward(dq, dk, pos, q=q, k=k, q_weight=w, k_weight=w)
    f = lambda q, w: (rot(q, k, pos, q_weight=w, k_weight=w)[0].double() * dq.double()).sum()
    h = 0.02
    for _ in range(4):
        d, e = torch.randn(q.shape, generator=gen).to(DEV), torch.randn(w.shape, generator=gen).to(DEV)
        diff = float((f(q + h * d, w) - f(q - h * d, w)) / (2 * h))
        size = float(got[0].abs().double().norm() * d.double().norm())
        assert abs(diff - float((got[0].double() * d.double()).sum())) < 2e-3 * size
        diff = float((f(q, w + h * e) - f(q, w - h * e)) / (2 * h))
        assert abs(diff - float((got[2].double() * e.double()).sum())) < 1e-4 * float(got[2].double().norm() * e.double().norm())


def test_positions_far_out_and_negative():
    rot = Rotary(64, layout="half", base=500000.0)
    pos = torch.tensor([0, 1, -1, 2 ** 20 + 1, 2 ** 31 - 1, -(2 ** 31), 2 ** 40 + 3, -(2 ** 50)])
    q = torch.randn(len(pos), 2, 64, generator=torch.Generator().manual_seed(7)).to(DEV)
    got, _ = rot(q, None, pos.to(DEV))
    # frequencies as the exact numbers that the operator holds: whole turns drop out of integer arithmetic
    turns = [t % 2 ** 64 for t in rot.turns.cpu().tolist()]
    angle = torch.tensor([[((int(p) * t) % 2 ** 64) / 2 ** 64 * 2 * math.pi for t in turns] for p in pos], dtype=torch.float64)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    x = q.double().cpu()
    want = torch.cat((x[..., :32] * c - x[..., 32:] * s, x[..., :32] * s + x[..., 32:] * c), -1)
    close(got, want, F32)
    # and for positions below 2^31 against the angle in 64 bits (53 bits of position * frequency: 2^-22 rad)
    near = plain64.rotate(x[:6], pos[None, :6], rot.frequencies, [0] * 32, layout="half")
    close(got[:6], near, F32)


def test_rows_of_zeros_infinities_and_nan():
    """A row of zeros stays zero under the norm; a NaN or an infinity reaches its own row (or head) and pair only."""
    rot = Rotary(32)
    q = torch.randn(5, 4, 32, generator=torch.Generator().manual_seed(8)).to(DEV)
    clean, _ = rot(q, None, torch.arange(5, device=DEV))
    q[1] = 0
    q[2, 1, 3] = math.nan
    q[3, 2, 8] = math.inf
    plain, _ = rot(q, None, torch.arange(5, device=DEV))
    bad = ~plain.isfinite()
    assert bad.sum() <= 4 and bool(bad[2, 1, 2:4].all()) and bool(bad[3, 2, 8:10].any())
    assert torch.equal(plain[[0, 4]], clean[[0, 4]]) and not bool(plain[1].any())
    for norm in (32, 128):
        got, _ = rot(q, None, torch.arange(5, device=DEV), q_weight=torch.ones(norm, device=DEV))
        assert not bool(got[1].any()) and bool(got[[0, 4]].isfinite().all())
        assert bool(got[2, 1].isnan().all()) and bool(got[2, 0].isfinite().all()) == (norm == 32)


def test_empty_and_single():
    rot = Rotary(128)
    q = torch.empty(0, 12, 128, dtype=BF, device=DEV)
    w = torch.ones(128, dtype=BF, device=DEV)
    got, none = rot(q, None, torch.empty(0, dtype=torch.int64, device=DEV))
    assert got.shape == q.shape and none is None
    back = rot.backward(q, q, torch.empty(0, dtype=torch.int64, device=DEV), q=q, k=q, q_weight=w, k_weight=w)
    assert back[0].shape == q.shape and not bool(back[2].any()) and not bool(back[3].any())


def test_offsets_beyond_32_bits():
    """2.2e9 elements, in place: the last tokens are as those of a small tensor."""
    N, H = 210011, 80
    rot = Rotary(128)
    q = torch.zeros(N, H, 128, dtype=BF, device=DEV)
    tail = torch.randn(3, H, 128, generator=torch.Generator().manual_seed(9)).to(BF).to(DEV)
    q[-3:] = tail
    pos = torch.arange(N, device=DEV)
    want, _ = rot(tail, None, pos[-3:])
    rot(q, None, pos, out=(q, None))
    assert torch.equal(q[-3:], want) and not bool(q[:2].any())


def test_yarn_and_bands_scale_cosine_and_frequencies():
    s = dict(type="yarn", factor=4.0, original_length=4096)
    rot = Rotary(128, layout="half", scaling=s)
    assert math.isclose(rot.mscale, 0.1 * math.log(4.0) + 1)
    q = torch.randn(7, 2, 128, generator=torch.Generator().manual_seed(10)).to(DEV)
    pos = torch.arange(7) + 5000
    got, _ = rot(q, None, pos.to(DEV))
    close(got, plain64.rotate(q.double().cpu(), pos[None], rot.frequencies, [0] * 64, layout="half", mscale=rot.mscale), F32)


def test_refusals():
    rot = Rotary(128, axes=(44, 42, 42))
    q = torch.zeros(4, 2, 128, dtype=BF, device=DEV)
    pos = torch.zeros(3, 4, dtype=torch.int64, device=DEV)
    w = torch.ones(128, dtype=BF, device=DEV)
    ok = dict(q_weight=w, k_weight=w)
    for call in (
        lambda: rot(q.cpu(), None, pos), lambda: rot(q.double(), None, pos), lambda: rot(q[..., :64], None, pos),
        lambda: rot(q, q.float(), pos), lambda: rot(q, q[:3], pos), lambda: rot(q, q.unsqueeze(0), pos),
        lambda: rot(q, None, pos[0]), lambda: rot(q, None, pos[:, :3]), lambda: rot(q, None, pos.float()),
        lambda: rot(q, None, pos.cpu()), lambda: rot(q, q, pos, q_weight=w), lambda: rot(q, q, pos, k_weight=w),
        lambda: rot(q, q, pos, q_weight=w[:64], k_weight=w), lambda: rot(q, q, pos, q_weight=w.half(), k_weight=w.half()),
        lambda: rot(q, q, pos, q_weight=torch.ones(256, dtype=BF, device=DEV), k_weight=w),
        lambda: rot(q, q, pos, inverse=True, **ok), lambda: rot(q, q, pos, out=(q, None)),
        lambda: rot(q, q, pos, out=(q, q[:2])), lambda: rot(q.transpose(1, 2).contiguous().transpose(1, 2), None, pos),
        lambda: rot.backward(q, q, pos, **ok), lambda: rot.backward(q, q, pos, q=q, **ok),
        lambda: rot.backward(q, q, pos, q=q, k=q[:3], **ok),
    ):
        with pytest.raises(ValueError):
            call()
    big = torch.zeros(1, 512, 128, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="exceeds"):
        rot.backward(big, big, pos[:, :1], q=big, k=big, **ok)


@pytest.mark.parametrize("case", [
    (9, 5, 5, 80, 40, "interleaved", None, "row", BF, True, 0),
    (333, 7, 2, 80, 40, "interleaved", (16, 12, 12), "head", F16, True, 5),
    (1200, 12, 3, 64, 24, "interleaved", None, "row", BF, False, 70000),
    (41, 3, 3, 48, 8, "interleaved", None, "", F16, False, 5),
    (90, 3, 1, 72, 36, "interleaved", None, "head", F32, True, 5),
    (3, 300, 2, 80, 40, "interleaved", None, "row", BF, False, 1),      # more heads than a block holds items of
], ids=str)
def test_rotated_part_of_whole_vectors(case):
    """The rotated part ends at a vector, but not at a pair of them."""
    test_forward_and_gradient(case, 0)
    test_forward_and_gradient(case, 2)


@pytest.mark.parametrize("norm", ["", "head", "row"])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("keys", [0, 3])
def test_autograd(norm, dtype, keys):
    """Gradients through torch.autograd are those of backward, with gradients of any strides; nothing is cut off silently."""
    gen = torch.Generator().manual_seed(12)
    rot = Rotary(64, 32, layout="half")
    pos = torch.arange(9, device=DEV) + 100
    q, k = make((9, 6, 64), dtype, gen, True, 3)
    k = k if keys else None
    dq, dk = make((9, 6, 64), dtype, gen, False, 3)
    w = [None, None]
    if norm:
        w = [(1 + 0.2 * torch.randn(n, generator=gen)).to(dtype).to(DEV) for n in ((64, 64) if norm == "head" else (6 * 64, 3 * 64))]
    if not keys:
        w[1] = None
    want = rot.backward(dq, dk if keys else None, pos, q=q, k=k, q_weight=w[0], k_weight=w[1])
    leaf = [None if t is None else t.detach().clone().requires_grad_() for t in (q, k, *w)]
    outs = rot(leaf[0], leaf[1], pos, q_weight=leaf[2], k_weight=leaf[3])
    assert torch.equal(outs[0], rot(q, k, pos, q_weight=w[0], k_weight=w[1])[0])
    torch.autograd.backward([t for t in outs if t is not None], [dq, dk][:1 + bool(keys)])
    for x, g in zip(leaf, want):
        assert (x is None) == (g is None) and (x is None or torch.equal(x.grad, g.to(x.dtype)))
    # an expanded gradient, one output alone, and one input or weight alone
    x = q.detach().clone().requires_grad_()
    rot(x, k, pos, q_weight=w[0], k_weight=w[1])[0].sum().backward()
    ones = rot.backward(torch.ones_like(q), None if k is None else torch.zeros_like(k), pos, q=q, k=k, q_weight=w[0], k_weight=w[1])
    assert torch.equal(x.grad, ones[0])
    if norm:
        x = w[0].detach().clone().requires_grad_()
        rot(q, k, pos, q_weight=x, k_weight=w[1])[0].backward(dq)
        assert torch.equal(x.grad, rot.backward(dq, None if k is None else torch.zeros_like(k), pos, q=q, k=k, q_weight=w[0],
                                                k_weight=w[1])[2].to(dtype))
    else:
        x = q.detach().clone().requires_grad_()
        rot(x, k, pos, inverse=True)[0].backward(dq)
        assert torch.equal(x.grad, rot(dq, None, pos)[0])
    with torch.no_grad():
        assert not rot(leaf[0], None, pos)[0].requires_grad


def test_writing_to_out_is_seen_by_autograd():
    rot = Rotary(64)
    pos = torch.arange(5, device=DEV)
    q, k = make((5, 4, 64), F32, torch.Generator().manual_seed(13), False, 4)
    w = torch.rand(64, device=DEV, requires_grad=True)
    loss = (q * w).sum()      # saves q
    rot(q, k, pos, out=(q, k))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    dq, dk, one = torch.ones_like(q), torch.ones_like(k), torch.ones(64, device=DEV)
    loss = (dq * w).sum()
    rot.backward(dq, dk, pos, q=q, k=k, q_weight=one, k_weight=one, out=(dq, dk))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    for kw in (dict(out=(torch.empty_like(q), torch.empty_like(k)), q_weight=w, k_weight=w),
               dict(out=(torch.empty_like(q).requires_grad_(), torch.empty_like(k)))):
        with pytest.raises(ValueError, match="requires a gradient"):
            rot(q, k, pos, **kw)
    with torch.inference_mode():
        x, y = q.clone(), k.clone()
        assert rot(x, y, pos, out=(x, y))[0] is x


@pytest.mark.parametrize("norm", ["", "head", "row"])
def test_no_heads_of_queries(norm):
    """k is turned all the same."""
    gen = torch.Generator().manual_seed(14)
    rot = Rotary(64)
    pos = torch.arange(7, device=DEV) + 3
    k, dk = make((7, 3, 64), F32, gen, False, 3)
    q = torch.empty(7, 0, 64, device=DEV)
    n = dict(head=64, row=3 * 64).get(norm)
    w = None if n is None else 1 + 0.2 * torch.randn(n, generator=gen).to(DEV)
    wq = None if n is None else torch.ones(64 if norm == "head" else 0, device=DEV)
    out = torch.full_like(k, 7.0)
    got = rot(q, k, pos, q_weight=wq, k_weight=w, out=(q, out))
    assert got[0] is q and got[1] is out and torch.equal(out, rot(k, None, pos, q_weight=w)[0])
    back = rot.backward(q, dk, pos, q=q, k=k, q_weight=wq, k_weight=w)
    want = rot.backward(dk, None, pos, q=k, q_weight=w)
    assert back[0].shape == q.shape and torch.equal(back[1], want[0])
    if norm:
        assert not bool(back[2].any()) and torch.equal(back[3], want[2])


@pytest.mark.parametrize("axes", [None, (24, 20, 20)])
@pytest.mark.parametrize("norm", ["", "row"])
def test_positions_shared_over_a_batch(axes, norm):
    """[N] or [A, N] for q [B, N, H, D], also as expanded, transposed and 32-bit views: as the sequences one by one."""
    gen = torch.Generator().manual_seed(15)
    rot = Rotary(64, layout="half", axes=axes)
    q, k = make((3, 11, 4, 64), BF, gen, True, 2)
    dq, dk = make((3, 11, 4, 64), BF, gen, False, 2)
    pos = (torch.randint(0, 5000, (11,) if axes is None else (3, 11), generator=gen)).to(DEV)
    w = (None, None) if not norm else tuple((1 + 0.2 * torch.randn(h * 64, generator=gen)).to(BF).to(DEV) for h in (4, 2))
    kw = dict(q_weight=w[0], k_weight=w[1])
    want = [rot(q[b], k[b], pos, **kw) for b in range(3)]
    grads = [rot.backward(dq[b], dk[b], pos, q=q[b], k=k[b], **kw) for b in range(3)]
    each = pos.unsqueeze(-2).expand(*pos.shape[:-1], 3, 11)
    for p in (pos, each, each.contiguous(), pos.to(torch.int32), pos.repeat_interleave(2, -1)[..., ::2]):
        got, back = rot(q, k, p, **kw), rot.backward(dq, dk, p, q=q, k=k, **kw)
        for i in range(2):
            assert torch.equal(got[i], torch.stack([t[i] for t in want])) and torch.equal(back[i], torch.stack([t[i] for t in grads]))


@pytest.mark.parametrize("dtype,D,rd", [(BF, 128, 128), (F16, 128, 64), (F32, 128, 128), (BF, 80, 40)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", ["", "head", "row"])
def test_addresses_that_are_not_whole_vectors(dtype, D, rd, layout, norm):
    """q, k, their gradients, results and weights at odd elements and odd strides, one at a time and all: what aligned copies give, but for
    the order of the norm's sums."""
    gen = torch.Generator().manual_seed(16)
    rot = Rotary(D, rd, layout=layout)
    N, H, Hk = 70, 5, 3
    pos = torch.arange(N, device=DEV) + 17
    q, k = make((N, H, D), dtype, gen, False, Hk)
    dq, dk = make((N, H, D), dtype, gen, False, Hk)
    w = [None, None] if not norm else [(1 + 0.2 * torch.randn(h * D if norm == "row" else D, generator=gen)).to(dtype).to(DEV) for h in (H, Hk)]
    off = {"x": (q, k), "dy": (dq, dk), "w": w}

    def odd(t, by):      # the same values `by` elements behind an aligned address, rows an odd number of elements apart
        if t is None:
            return None
        if t.dim() == 1:
            base = torch.empty(len(t) + by, dtype=t.dtype, device=DEV)
            base[by:] = t
            return base[by:]
        n, h, d = t.shape
        base = torch.empty(by + n * (h * (d + 1) + 1), dtype=t.dtype, device=DEV)
        view = base[by:].as_strided((n, h, d), (h * (d + 1) + 1, d + 1, 1), by)
        return view.copy_(t)

    args, weights = (pos[None].cpu(), rot.frequencies, axis_of(rot)), [None if t is None else t.cpu() for t in w]
    exact = [plain64.rotary(t.double().cpu(), v, 1e-6, *args, layout=layout) for t, v in zip((q, k), weights)]
    exact_grad = [plain64.rotary_grad(d.double().cpu(), t.double().cpu(), v, 1e-6, *args, layout=layout)[0]
                  for d, t, v in zip((dq, dk), (q, k), weights)]
    for by in (1, 3):
        for which in ("x", "dy", "w", "out", "all"):
            use = {n: [odd(t, by) if which in (n, "all") else t for t in ts] for n, ts in off.items()}
            out = tuple(odd(t, by) if which in ("out", "all") else torch.empty_like(t) for t in (q, k))
            got = rot(*use["x"], pos, q_weight=use["w"][0], k_weight=use["w"][1], out=out)
            for g, e in zip(got, exact):
                close(g, e, dtype)
            back = rot.backward(*use["dy"], pos, q=use["x"][0], k=use["x"][1], q_weight=use["w"][0], k_weight=use["w"][1], out=out)
            for g, e in zip(back, exact_grad):
                close(g, e, dtype)
