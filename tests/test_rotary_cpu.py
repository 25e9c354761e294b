"""Rotary positions without a GPU: frequencies, plans, refusals of the C entry, and the gradient's formula against
differences of the definition in 64 bits."""
import ctypes
import math

import pytest
import torch

import plain64
from token2tile_b200 import Rotary, latent_positions, rotary_frequencies


def test_frequencies():
    f, m = rotary_frequencies(8, 10000.0)
    assert m == 1.0 and all(math.isclose(a, b) for a, b in zip(f, (1.0, 0.1, 0.01, 0.001)))
    assert rotary_frequencies(8, scaling=dict(type="linear", factor=2.0))[0] == [x / 2 for x in f]
    n, _ = rotary_frequencies(8, scaling=dict(type="ntk", factor=4.0))
    assert math.isclose(n[0], f[0]) and math.isclose(n[-1], f[-1] / 4)
    for kind in ("yarn", "bands"):
        y, m = rotary_frequencies(128, scaling=dict(type=kind, factor=4.0, original_length=4096))
        g, _ = rotary_frequencies(128)
        assert math.isclose(y[0], g[0]) and math.isclose(y[-1], g[-1] / 4)
        assert all(b / 4 - 1e-18 <= a <= b for a, b in zip(y, g))
        assert math.isclose(m, 0.1 * math.log(4.0) + 1 if kind == "yarn" else 1.0)


def test_plan_holds_frequencies_as_turns():
    rot = Rotary(128, axes=(44, 42, 42), device="cpu")
    assert rot.axis.tolist() == [0] * 22 + [1] * 21 + [2] * 21
    for t, f in zip(rot.turns.tolist(), rot.frequencies):
        assert math.isclose((t % 2 ** 64) / 2 ** 64, f / (2 * math.pi) % 1.0, rel_tol=1e-15)


def test_latent_positions():
    p = latent_positions(2, 3, 4, device="cpu")
    assert p.shape == (3, 24) and p[:, 0].tolist() == [0, 0, 0] and p[:, 23].tolist() == [1, 2, 3] and p[:, 5].tolist() == [0, 1, 1]
    assert torch.equal(latent_positions(2, 3, 4, start=7, count=9, device="cpu"), p[:, 7:16])


def test_refusals():
    for args in ((0,), (127,), (128, 130), (128, 3), (1024, 1024)):
        with pytest.raises(ValueError):
            Rotary(*args, device="cpu")
    for kw in (dict(layout="pairs"), dict(axes=(64, 32)), dict(axes=(63, 65)), dict(base=0.0),
               dict(scaling=dict(type="stretch", factor=2.0)), dict(scaling=dict(type="linear", factor=-1.0)),
               dict(scaling=dict(type="linear", factor=2.0, original_length=3))):
        with pytest.raises(ValueError):
            Rotary(128, device="cpu", **kw)


def test_entry_points_refuse_bad_arguments(lib):
    x = 4096                     # never read: every call is refused before anything is launched
    strides = (ctypes.c_longlong * 18)(*[128] * 18)
    s = ctypes.addressof(strides)

    def call(q=x, out=x, pos=x, bytes_=8, batch=1, N=4, H=2, Hk=2, D=128, rd=128, inverse=0, norm=0, w=0, dtype=0, wd=0):
        return lib.t2t_rotary(q, x, out, x, w, w, wd, pos, bytes_, 0, 0, x, x, s, batch, N, H, Hk, D, rd, 1, inverse, norm, 1.0,
                              1e-6, dtype, 0)

    for kw in (dict(q=0), dict(out=0), dict(pos=0), dict(bytes_=2), dict(batch=0), dict(N=0), dict(H=0), dict(Hk=-1), dict(D=127),
               dict(rd=0), dict(rd=130), dict(rd=5), dict(D=2048, rd=1024), dict(norm=3, w=x), dict(norm=1), dict(norm=2, w=x, inverse=1),
               dict(dtype=3), dict(wd=1), dict(batch=1 << 20, N=1 << 20)):
        assert call(**kw) == 1, kw

    def grad(norm=1, ws=x, ws_bytes=1 << 30, H=2, D=128, dw=x):
        return lib.t2t_rotary_grad(x, x, x, x, x, x, x, x, 0, dw, x, x, 8, 0, 0, x, x, s, 1, 4, H, 2, D, 2, 1, norm, 1.0, 1e-6, 0, ws,
                                   ws_bytes, 0)

    assert grad(norm=0) == 1 and grad(ws=0) == 1 and grad(dw=0) == 1
    assert grad(ws_bytes=lib.t2t_rotary_grad_ws_bytes(2, 2, 128, 1) - 1) == 3
    assert grad(H=400) == 4


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("norm", ["", "head", "row"])
def test_gradient_formula_against_differences(layout, norm):
    """Central differences of the definition in 64 bits, h = 1e-5: off by h^2 and 1e-16 / h."""
    gen = torch.Generator().manual_seed(3)
    x, dy = (torch.randn(3, 2, 8, generator=gen, dtype=torch.float64) for _ in range(2))
    w = None if not norm else 1 + 0.3 * torch.randn(16 if norm == "row" else 8, generator=gen, dtype=torch.float64)
    pos = torch.tensor([[0, 5, 17]])
    args, kw = (pos, [1.0, 0.1, 0.01], [0, 0, 0]), dict(layout=layout, mscale=1.25)
    f = lambda x, w: (plain64.rotary(x, w, 1e-6, *args, **kw) * dy).sum()
    dx, dw = plain64.rotary_grad(dy, x, w, 1e-6, *args, **kw)
    h = 1e-5
    for i in range(x.numel()):
        d = torch.zeros_like(x)
        d.view(-1)[i] = h
        assert abs(float((f(x + d, w) - f(x - d, w)) / (2 * h) - dx.view(-1)[i])) < 1e-8
    for i in range(0 if w is None else w.numel()):
        d = torch.zeros_like(w)
        d[i] = h
        assert abs(float((f(x, w + d) - f(x, w - d)) / (2 * h) - dw[i])) < 1e-8


def test_yarn_attention_factor():
    """0.1 ln(factor) + 1 for stretched contexts, 1 where nothing is stretched, or as given."""
    of = lambda factor, **kw: rotary_frequencies(64, scaling=dict(type="yarn", factor=factor, original_length=4096, **kw))[1]
    assert math.isclose(of(8.0), 0.1 * math.log(8.0) + 1) and of(1.0) == of(0.5) == of(0.01) == 1.0
    assert of(0.5, attention_factor=0.7) == 0.7


def test_refuses_tensors_on_the_host():
    """A plan made on the host has the host's tensors pass as its own; their pointers never reach a kernel."""
    rot = Rotary(8, device="cpu")
    q, pos, w = torch.zeros(2, 3, 8), torch.arange(2), torch.ones(8)
    for call in (lambda: rot(q, None, pos), lambda: rot(q, q, pos, q_weight=w, k_weight=w), lambda: rot.backward(q, None, pos),
                 lambda: rot.backward(q, q, pos, q=q, k=q, q_weight=w, k_weight=w)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_error_of_the_frequencies():
    """The frequencies are 64-bit floats, turned into turns in 64-bit floats: within 2^-55 turns a position of the exact f / (2 pi), which is
    what limits the angle far out (behind 2^29 positions it is more than the rounding to 32 bits).  That whole turns drop out
    exactly says nothing about this."""
    from fractions import Fraction
    pi = Fraction(31415926535897932384626433832795028841971693993751058209749445923, 10 ** 64)
    for width, base in ((8, 1e4), (64, 1e4), (128, 5e5), (128, 1e6), (256, 1e4), (512, 1e4)):
        rot = Rotary(width, base=base, device="cpu")
        for t, f in zip(rot.turns.tolist(), rot.frequencies):
            off = abs(Fraction(t % 2 ** 64, 2 ** 64) - Fraction(f) / (2 * pi))
            assert off <= Fraction(1, 2 ** 55)


def test_refusals_of_scalings():
    for kind in ("yarn", "bands"):
        for kw in (dict(), dict(original_length=0), dict(original_length=-4096)):
            with pytest.raises(ValueError, match="original_length"):
                rotary_frequencies(64, scaling=dict(type=kind, factor=2.0, **kw))
    with pytest.raises(ValueError, match="base"):
        rotary_frequencies(64, 1.0, scaling=dict(type="yarn", factor=2.0, original_length=4096))
    assert rotary_frequencies(64, 1.0)[0] == [1.0] * 32
