"""4-bit quantisation, products and layers against their definitions in 64 bits.

Quantisation is exact where no arithmetic stands in front of it: codes and scales have to be equal.  Products: the operands'
products are exact in 32 bits; adding K of them in 32 bits, in any order and with truncation instead of rounding, is off by at most
K 2^-23 of the sum of their magnitudes; the activation (2^-20 relative), bias, gate and residual add a few 2^-23 of the same sum,
and the result is rounded once (2^-8, 2^-11, 2^-23 of it)."""
import math

import pytest
import torch

import plain64
from token2tile_b200 import Fp4FeedForward, Fp4Linear, Fp4Tensor, fp4_matmul, fp4_quantize, fp4_tensor_scale
from token2tile_b200.fp4 import check_status

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ULP = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -23}
FMTS = ("mxfp4", "nvfp4")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def codes_of(t):
    """Codes 0 .. 15 [M, K] and scale bytes [M, blocks] of an Fp4Tensor, read from its layout as the C header describes it."""
    M, K = t.shape
    c = t.codes.cpu()
    codes = torch.stack((c & 15, c >> 4), -1).flatten(1)
    assert not bool(codes[:, K:].any())                       # zeros behind the last element
    blocks = -(-K // plain64.BLOCK[t.fmt])
    atoms = -(-blocks // 4)
    s = t.scales.cpu()
    r, b = torch.arange(M)[:, None], torch.arange(4 * atoms)[None]
    scales = s[((r // 128) * atoms + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4]
    assert not bool(scales[:, blocks:].any())                 # and behind the last block
    return codes[:, :K].long(), scales[:, :blocks]


def scale_values(b, fmt):
    if fmt == "nvfp4":
        return b.view(torch.float8_e4m3fn).double()
    return torch.where(b == 255, math.nan, torch.ldexp(torch.ones(b.shape, dtype=torch.float64), b.int() - 127))


def check_quantized(t, x, g=1.0):
    code, scale, value = plain64.quantize(x.double().cpu(), t.fmt, g)
    got_code, got_scale = codes_of(t)
    assert torch.equal(scale_values(got_scale, t.fmt).nan_to_num(-1.0), scale.nan_to_num(-1.0))
    ok = ~value.isnan()
    zero = value == 0                                           # the sign of a zero is free
    assert torch.equal((got_code & 7)[ok], (code & 7)[ok]) and torch.equal(got_code[ok & ~zero], code[ok & ~zero])
    back = t.dequantize(F32).cpu().double()
    assert torch.equal(back.isnan(), value.isnan()) and torch.equal(back[ok], value[ok])


def tricky(M, K, dtype, seed):
    """Normal values with outliers, zeros, whole blocks of zeros, ties, and magnitudes far apart."""
    g = gen(seed)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-12, 12, (M, 1), generator=g).float())
    x = torch.where(torch.rand(M, K, generator=g) < 0.05, 0.0, x)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.5, 7.0, 7.9, 4.0])
    rows = torch.arange(M) % 3 == 1
    pick = ties[torch.randint(0, len(ties), (M, K), generator=g)] * torch.exp2(torch.randint(-6, 7, (M, 1), generator=g).float())
    # times the possible significands of a block's scale
    pick = pick * (1 + torch.randint(0, 8, (M, 1), generator=g) / 8)
    x = torch.where(rows[:, None], pick * torch.where(torch.rand(M, K, generator=g) < 0.5, -1.0, 1.0), x)
    x[:, :K // 3][torch.arange(M) % 5 == 2] = 0
    return x.to(dtype)


SHAPES = [(1, 1), (1, 16), (2, 17), (3, 31), (5, 32), (7, 33), (4, 64), (130, 100), (129, 1000), (257, 513), (33, 5120)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,K", SHAPES)
def test_quantize(fmt, dtype, M, K):
    x = tricky(M, K, dtype, M * 7 + K)
    check_quantized(fp4_quantize(x.to(DEV), fmt), x)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_every_tie_of_every_scale(dtype):
    """nvfp4: the middles between codes times every significand a block's scale can have, with 6 times the scale as the block's
    largest magnitude: all of them exact in every type."""
    rows = []
    for m in range(8):
        for e in (-6, -3, 0, 4):
            s = (1 + m / 8) * 2.0 ** e
            rows.append([6 * s, 0.25 * s, 0.75 * s, -1.25 * s, 1.75 * s, -2.5 * s, 3.5 * s, 5 * s] + [0.0] * 8)
    x = torch.tensor(rows, dtype=torch.float64)
    assert torch.equal(x.to(dtype).double(), x)
    t = fp4_quantize(x.to(dtype).to(DEV), "nvfp4")
    check_quantized(t, x)
    assert codes_of(t)[0][:, :8].tolist() == [[7, 0, 2, 10, 4, 12, 6, 6]] * len(rows)


def test_neighbours_of_ties():
    """32-bit elements one unit in the last place above and below every middle between codes, under every significand of a scale."""
    rows = []
    for m in range(8):
        s = (1 + m / 8) * 0.5
        mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]) * s
        up, down = torch.nextafter(mid, torch.tensor(math.inf)), torch.nextafter(mid, torch.tensor(0.0))
        rows.append(torch.cat((torch.tensor([6 * s]), mid, up, torch.zeros(1), torch.tensor([6 * s]), down, -up, torch.zeros(1))))
    x = torch.stack(rows)
    check_quantized(fp4_quantize(x.to(DEV), "nvfp4"), x)
    x = torch.randn(512, 4096, generator=gen(3))
    check_quantized(fp4_quantize(x.to(DEV), "nvfp4"), x)


@pytest.mark.parametrize("g", [2.0 ** -9, 2.0 ** 3, 2.0 ** -100, 2.0 ** 90])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_tensor_scale(g, dtype):
    x = tricky(64, 200, dtype, 5)
    t = fp4_quantize(x.to(DEV), "nvfp4", tensor_scale=g)
    assert t.tensor_scale == g
    check_quantized(t, x, g)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_extremes(fmt, dtype):
    """Blocks of the largest and the smallest numbers, zeros of both signs, infinities and NaN: these make their own block NaN."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(9, 96)
    x[0] = big
    x[1] = -big
    x[2] = tiny
    x[3] = tiny / 4                                             # subnormal
    x[4] = -0.0
    x[5, 5], x[5, 40] = math.inf, 1.0
    x[6, 70], x[6, 0] = math.nan, 3.0
    x[7, 0], x[7, 1] = 448 * 6.0, 1.0
    x[8, 3], x[8, 17] = 1e-3, -math.inf
    x = x.to(dtype)
    t = fp4_quantize(x.to(DEV), fmt)
    check_quantized(t, x)


def test_strided_rows_and_leading_dimensions():
    base = torch.randn(6, 10, 72, generator=gen(11)).to(BF).to(DEV)
    for x in (base[:, 0], base[:, 3, 8:], base[:, 5, 1:65], base, base[:, :, :64], base[2:, 0, :1], base[:, 1, 3:], base[:, 2, 5:70]):
        t = fp4_quantize(x)
        check_quantized(t, x.reshape(-1, x.shape[-1]))
    odd = torch.randn(9, 91, generator=gen(12)).to(DEV)
    for x in (odd, odd[:, 1:], odd[1:, 2:50], odd[:, 3:40]):
        check_quantized(fp4_quantize(x), x)
        out = torch.full((9, 95), 7.0, device=DEV)[:x.shape[0], 2:2 + x.shape[1]]
        fp4_quantize(x).dequantize(out=out)
        assert torch.equal(out, fp4_quantize(x).dequantize())
    with pytest.raises(ValueError):
        fp4_quantize(base[:, :5])
    with pytest.raises(ValueError):
        fp4_quantize(base.transpose(1, 2))


@pytest.mark.parametrize("fmt", FMTS)
def test_stored_form(fmt):
    for M, K in ((1, 1), (3, 33), (130, 100), (300, 256)):
        b = plain64.BLOCK[fmt]
        packed = torch.randint(0, 256, (M, -(-K // 2)), generator=gen(M), dtype=torch.uint8)
        scales = torch.randint(40, 120, (M, -(-K // b)), generator=gen(K), dtype=torch.uint8)
        if K % 2:
            packed[:, -1] &= 15
        t = Fp4Tensor.from_stored(packed.to(DEV), scales.to(DEV), K, fmt, tensor_scale=0.5)
        codes, got = codes_of(t)
        assert torch.equal(got, scales)
        assert torch.equal(codes, torch.stack((packed & 15, packed >> 4), -1).flatten(1)[:, :K].long())
        p, s = t.to_stored()
        assert torch.equal(p.cpu(), packed) and torch.equal(s.cpu(), scales)
        v = torch.copysign(plain64.VALUES[codes & 7], 7.5 - codes) * scale_values(scales, fmt).repeat_interleave(b, 1)[:, :K] * 0.5
        assert torch.equal(t.dequantize(F32).cpu().double(), v.float().double())
        assert torch.equal(t.dequantize(BF).cpu(), v.to(BF))
    kinds = dict(mxfp4=torch.float8_e4m3fn, nvfp4=torch.float8_e8m0fnu)
    with pytest.raises(ValueError):
        Fp4Tensor.from_stored(packed.to(DEV), scales.to(DEV).view(kinds[fmt]), K, fmt)


def stored(M, K, fmt, seed, spread=3):
    b = plain64.BLOCK[fmt]
    packed = torch.randint(0, 256, (M, -(-K // 2)), generator=gen(seed), dtype=torch.uint8)
    lo, hi = (127 - spread, 127 + spread) if fmt == "mxfp4" else (56 - 8 * spread, 56 + 8 * spread)
    scales = torch.randint(lo, hi, (M, -(-K // b)), generator=gen(seed + 1), dtype=torch.uint8)
    return Fp4Tensor.from_stored(packed.to(DEV), scales.to(DEV), K, fmt)


def values(t):
    return t.dequantize(F32).cpu().double()


def check_product(got, a, w, dtype, **kw):
    K = a.shape[1]
    want, size = plain64.matmul(values(a), values(w), a.tensor_scale * 0 + 1.0, **kw)
    err = (got.cpu().double() - want).abs()
    tol = ULP[dtype] * want.abs() + (K + 16) * 2.0 ** -23 * size + (2.0 ** -25 if dtype == F16 else 1e-30)
    assert bool((err <= tol).all()), (float((err / tol).max()), int((err > tol).sum()), err.shape)


MM_SHAPES = [(1, 1, 1), (1, 16, 16), (1, 300, 513), (2, 128, 64), (3, 129, 100), (8, 257, 320), (17, 65, 1000), (33, 512, 96),
             (64, 40, 2048), (100, 384, 272), (127, 127, 127), (128, 128, 256), (129, 130, 258), (200, 1000, 160), (256, 256, 512),
             (257, 513, 528), (300, 31, 64), (513, 260, 1040), (700, 1000, 304), (1, 4099, 4100),
             # more row tiles than SMs: pairs of CTAs, one and several tiles a pair
             (1300, 1930, 272), (260, 9500, 96), (2500, 1000, 528), (2049, 2055, 80), (5000, 4104, 64), (3000, 1025, 2080)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", MM_SHAPES)
def test_product(fmt, M, N, K):
    a, w = stored(M, K, fmt, M + N), stored(N, K, fmt, K + 1)
    check_product(fp4_matmul(a, w, dtype=F32), a, w, F32)
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("activation", [None, "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,N,K", [(1, 200, 128), (5, 264, 320), (140, 136, 96), (300, 520, 512), (1500, 1672, 96), (2100, 1287, 80)])
def test_epilogue(fmt, dtype, activation, M, N, K):
    a, w = stored(M, K, fmt, M + N), stored(N, K, fmt, K + 1)
    a.tensor_scale = 2.0 ** -round(0.5 * math.log2(K) + 4)
    g = gen(M)
    bias, gate = (torch.randn(N, generator=g).to(dtype) for _ in range(2))
    residual = torch.randn(M, N, generator=g).to(dtype)
    on = lambda t: t.to(DEV)
    kw = dict(bias=bias, activation=activation, gate=gate, residual=residual)
    got = fp4_matmul(a, w, dtype=dtype, **{k: v if isinstance(v, (str, type(None))) else on(v) for k, v in kw.items()})
    assert got.dtype == dtype
    check_product(got, a, w, dtype, **kw)
    for drop in ("bias", "gate", "residual"):
        part = {k: v for k, v in kw.items() if k != drop}
        got = fp4_matmul(a, w, dtype=dtype, **{k: v if isinstance(v, (str, type(None))) else on(v) for k, v in part.items()})
        check_product(got, a, w, dtype, **part)
    # 32-bit vectors beside any type; into the residual's storage, inside a wider matrix
    wide = torch.full((M, N + 24), 7.0, dtype=dtype, device=DEV)
    for off in (8, 3):
        wide.fill_(7.0)
        wide[:, off:off + N] = on(residual)
        view = wide[:, off:off + N]
        got = fp4_matmul(a, w, bias=on(bias).float(), activation=activation, gate=on(gate).float(), residual=view, out=view)
        assert got.data_ptr() == view.data_ptr()
        check_product(view, a, w, dtype, **kw)
        assert bool((wide[:, :off] == 7).all()) and bool((wide[:, off + N:] == 7).all())
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 20, 140, 300, 7000])
def test_nan_scales_reach_their_row_or_column_only(fmt, M):
    N, K = 300, 160
    x, y = torch.randn(M, K, generator=gen(1)), torch.randn(N, K, generator=gen(2))
    x[M // 2, 3] = math.nan
    y[7, 150], y[299, 0] = math.inf, math.nan
    got = fp4_matmul(fp4_quantize(x.to(DEV), fmt), fp4_quantize(y.to(DEV), fmt), dtype=F32)
    want = torch.zeros(M, N, dtype=torch.bool)
    want[M // 2], want[:, 7], want[:, 299] = True, True, True
    assert torch.equal(got.isnan().cpu(), want) and not bool(got.isinf().any())
    check_status()


@pytest.mark.parametrize("M", [1, 200, 600, 3001])
def test_same_bits_every_time_and_on_another_stream(M):
    a, w = stored(M, 2080, "nvfp4", 3), stored(1000, 2080, "nvfp4", 4)
    want = fp4_matmul(a, w, dtype=F32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            got = fp4_matmul(a, w, dtype=F32)
        side.synchronize()
        assert torch.equal(got, want)
    check_status()


def test_large_scales_and_cancelling_sums():
    """Scales at both ends of their range, and rows whose products cancel to a thousandth of their magnitudes."""
    for fmt in FMTS:
        a, w = stored(130, 512, fmt, 5), stored(140, 512, fmt, 6)
        lo, hi = (127 - 55, 127 + 55) if fmt == "mxfp4" else (1, 126)
        for t in (a, w):
            s = torch.randint(lo, hi + 1, (t.shape[0], 512 // plain64.BLOCK[fmt]), generator=gen(7), dtype=torch.uint8)
            p, _ = t.to_stored()
            u = Fp4Tensor.from_stored(p, s.to(DEV), 512, fmt)
            t.data = u.data
        check_product(fp4_matmul(a, w, dtype=F32), a, w, F32)
    x = torch.randn(130, 256, generator=gen(8)).to(DEV)
    a = fp4_quantize(torch.cat((x, -x), 1), "nvfp4")
    y = torch.randn(100, 256, generator=gen(9)).to(DEV)
    w = fp4_quantize(torch.cat((y, y), 1), "nvfp4")
    got = fp4_matmul(a, w, dtype=F32)
    check_product(got, a, w, F32)
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 48), (130, 256), (9, 1000), (5, 5120), (2, 13824), (3, 20000),
                                 (700, 1001), (1201, 333), (5, 20481), (2, 30001)])
def test_modulated_quantize(fmt, dtype, M, K):
    """The modulated norm is in 32 bits (1e-5 of the row's largest at worst), so a value next to a middle between codes may fall to
    either side: every value within one step of what is quantised, and all but one in a thousand equal."""
    g = gen(M + K)
    x = (torch.randn(M, K, generator=g) * 3 + torch.randn(M, 1, generator=g)).to(dtype)
    shift, scale = ((0.2 * torch.randn(K, generator=g)).to(dtype) for _ in range(2))
    t = fp4_quantize(x.to(DEV), fmt, shift=shift.to(DEV), scale=scale.to(DEV))
    y = plain64.modulated(x.double(), shift.double(), scale.double())
    _, s, value = plain64.quantize(y, fmt)
    got = values(t)
    step = (s.repeat_interleave(plain64.BLOCK[fmt], 1)[:, :K]) * 2 * 1.2
    # mxfp4: a largest magnitude next to a power of two may double or halve its block's scale
    assert bool(((got - y).abs() <= step * (2 if fmt == "mxfp4" else 1) + 1e-30).all())
    assert float((got != value).double().mean()) < 1e-3 + 40.0 / (M * K) * (M * K < 40000)


def test_modulated_rows_of_one_value():
    """No variance: eps keeps the reciprocal finite, what is quantised is the shift."""
    x = torch.full((3, 64), 5.0, dtype=BF, device=DEV)
    x[2] = 0
    shift, scale = torch.ones(64, dtype=BF, device=DEV), torch.zeros(64, dtype=BF, device=DEV)
    check_quantized(fp4_quantize(x, "nvfp4", shift=shift, scale=scale), torch.ones(3, 64))
    x[1, 3] = math.nan
    got = fp4_quantize(x, "nvfp4", shift=shift, scale=scale).dequantize(F32)
    assert bool(got[1].isnan().all()) and bool(got[[0, 2]].isfinite().all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 3, 150])
def test_linear(fmt, M):
    """From values that are quantised exactly, so that the layer is the product of known matrices."""
    g = gen(M)
    x = torch.randn(M, 2, 320, generator=g).to(BF)
    weight = (torch.randn(200, 320, generator=g) / 18).to(BF)
    bias = torch.randn(200, generator=g).to(BF)
    layer = Fp4Linear(weight.to(DEV), bias.to(DEV), fmt=fmt)
    gs = layer.w.tensor_scale
    assert fmt == "mxfp4" or gs == fp4_tensor_scale(weight)
    got = layer(x.to(DEV), activation="silu")
    assert got.shape == (M, 2, 200) and got.dtype == BF
    a = plain64.quantize(x.double().view(-1, 320), fmt)[2]
    w = plain64.quantize(weight.double(), fmt, gs)[2]
    want, size = plain64.matmul(a, w, bias=bias, activation="silu")
    err = (got.cpu().double().view(-1, 200) - want).abs()
    assert bool((err <= ULP[BF] * want.abs() + 336 * 2.0 ** -23 * size).all())
    out = torch.empty_like(got)
    assert layer(x.to(DEV), activation="silu", out=out) is out and torch.equal(out, got)
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [1, 70])
def test_feed_forward(fmt, M):
    """Against the layers one by one; a hidden value next to a middle between codes may fall to either side: one step of one of 384
    elements, 2e-2 of the output in the worst case, 2e-3 of its norm."""
    g = gen(M)
    x = torch.randn(M, 256, generator=g).to(BF).to(DEV)
    vec = lambda n: torch.randn(n, generator=g).to(BF).to(DEV) * 0.1
    up = Fp4Linear((torch.randn(384, 256, generator=g) / 16).to(BF).to(DEV), vec(384), fmt=fmt)
    down = Fp4Linear((torch.randn(256, 384, generator=g) / 20).to(BF).to(DEV), vec(256), fmt=fmt)
    shift, scale, gate = vec(256), vec(256), vec(256) + 0.5
    got = Fp4FeedForward(up, down)(x, shift=shift, scale=scale, gate=gate, residual=x)
    y = plain64.modulated(*(t.double().cpu() for t in (x, shift, scale)))
    h, _ = plain64.matmul(plain64.quantize(y, fmt)[2], values(up.w), bias=up.b.cpu(), activation="gelu_tanh")
    want, _ = plain64.matmul(plain64.quantize(h, fmt)[2], values(down.w), bias=down.b.cpu(), gate=gate.cpu(), residual=x.cpu())
    err = got.cpu().double() - want
    assert float(err.norm() / (want - x.double().cpu()).norm()) < 1e-2
    assert float(err.abs().max()) < 0.1
    # one call for what the operators do one by one
    a = fp4_quantize(x, fmt, shift=shift, scale=scale)
    h = fp4_matmul(a, up.w, bias=up.b, activation="gelu_tanh", dtype=fmt)
    assert torch.equal(got, fp4_matmul(h, down.w, bias=down.b, gate=gate, residual=x))
    out = x.clone().view(M, 1, 256)
    assert Fp4FeedForward(up, down)(out, shift=shift, scale=scale, gate=gate, residual=out, out=out) is out
    assert torch.equal(out.view(M, 256), got)
    for bad in (dict(shift=shift), dict(gate=gate[:9]), dict(residual=x[:, :9]), dict(out=x.float())):
        with pytest.raises(ValueError):
            Fp4FeedForward(up, down)(x, **bad)
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 64), (1, 5120, 96), (3, 40, 160), (20, 333, 64), (140, 1000, 272), (300, 72, 64),
                                   (257, 513, 64), (1500, 1700, 96), (2100, 1287, 272), (300, 9000, 64)])
def test_quantised_product(fmt, M, N, K):
    """The result in 32 bits, quantised: bit for bit what quantising the 32-bit result of the same product gives."""
    a, w = stored(M, K, fmt, M), stored(N, K, fmt, N)
    a.tensor_scale = 2.0 ** -round(0.5 * math.log2(K) + 4)
    bias, gate = (torch.randn(N, generator=gen(i)).to(DEV) for i in (1, 2))
    for kw in (dict(), dict(bias=bias, activation="gelu_tanh", gate=gate)):
        want = fp4_quantize(fp4_matmul(a, w, dtype=F32, **kw), fmt)
        got = fp4_matmul(a, w, dtype=fmt, **kw)
        for x, y in zip(codes_of(got), codes_of(want)):
            assert torch.equal(x, y)
        out = Fp4Tensor.empty(M, N, fmt, 1.0 if fmt == "mxfp4" else 2.0 ** -3, DEV)
        assert fp4_matmul(a, w, out=out, **kw) is out
        want = fp4_quantize(fp4_matmul(a, w, dtype=F32, **kw), fmt, tensor_scale=out.tensor_scale)
        for x, y in zip(codes_of(out), codes_of(want)):
            assert torch.equal(x, y)
    check_status()


def test_empty():
    x = torch.empty(0, 64, dtype=BF, device=DEV)
    t = fp4_quantize(x)
    w = fp4_quantize(torch.ones(32, 64, dtype=BF, device=DEV))
    assert t.shape == (0, 64) and t.dequantize().shape == (0, 64) and fp4_matmul(t, w).shape == (0, 32)
    assert fp4_matmul(w, t).shape == (32, 0)
    assert Fp4Linear(w)(torch.empty(2, 0, 64, dtype=BF, device=DEV)).shape == (2, 0, 32)


def test_offsets_beyond_32_bits():
    """More than 2^31 elements in, and out of a product: the last rows are as those of a small matrix."""
    M, K = 450001, 5000
    x = torch.zeros(M, K, dtype=BF, device=DEV)
    tail = torch.randn(5, K, generator=gen(12)).to(BF).to(DEV)
    x[-5:] = tail
    t = fp4_quantize(x)
    del x
    codes, scales = t.to_stored()
    want, ws = fp4_quantize(tail).to_stored()
    assert torch.equal(codes[-5:], want) and torch.equal(scales[-5:], ws) and not bool(codes[:100].any())
    back = t.dequantize(BF)
    assert torch.equal(back[-5:], fp4_quantize(tail).dequantize(BF))
    del back, codes, scales
    M, N = 140003, 16390
    a, w = stored(M, 48, "nvfp4", 13), stored(N, 48, "nvfp4", 14)
    got = fp4_matmul(a, w)
    last = Fp4Tensor.from_stored(*(p[-300:] for p in a.to_stored()), 48, "nvfp4")
    assert torch.equal(got[-300:], fp4_matmul(last, w))
    check_status()


def test_refusals():
    x = torch.zeros(4, 64, dtype=BF, device=DEV)
    t, w = fp4_quantize(x), fp4_quantize(torch.zeros(32, 64, dtype=BF, device=DEV))
    v = torch.zeros(64, dtype=BF, device=DEV)
    b = torch.zeros(32, dtype=BF, device=DEV)
    r = torch.zeros(4, 32, dtype=BF, device=DEV)
    lin = Fp4Linear(w, b)
    for call in (
        lambda: fp4_quantize(x.cpu()), lambda: fp4_quantize(x.double()), lambda: fp4_quantize(x, "fp4"), lambda: fp4_quantize(x[:, :0]),
        lambda: fp4_quantize(x, tensor_scale=0.0), lambda: fp4_quantize(x, tensor_scale=math.nan),
        lambda: fp4_quantize(x, "mxfp4", tensor_scale=2.0), lambda: fp4_quantize(x, shift=v), lambda: fp4_quantize(x, scale=v),
        lambda: fp4_quantize(x, shift=v[:32], scale=v), lambda: fp4_quantize(x, shift=v.float(), scale=v),
        lambda: fp4_quantize(x, shift=v.cpu(), scale=v), lambda: fp4_quantize(x, out=w), lambda: fp4_quantize(x.t()),
        lambda: fp4_matmul(t, fp4_quantize(x[:, :32])), lambda: fp4_matmul(t, fp4_quantize(x, "mxfp4")),
        lambda: fp4_matmul(t, w, activation="relu"), lambda: fp4_matmul(t, w, bias=v), lambda: fp4_matmul(t, w, gate=b.cpu()),
        lambda: fp4_matmul(t, w, bias=b, gate=b.float()), lambda: fp4_matmul(t, w, residual=r[:3]),
        lambda: fp4_matmul(t, w, residual=r.float()), lambda: fp4_matmul(t, w, dtype="mxfp4"), lambda: fp4_matmul(t, w, out=t),
        lambda: fp4_matmul(t, w, dtype="nvfp4", residual=r), lambda: fp4_matmul(t, w, out=r.t()), lambda: fp4_matmul(t, w, dtype=torch.int32),
        lambda: lin(x[:, :32]), lambda: lin(x, residual=r[:2]), lambda: lin(x, out=r[:2]), lambda: Fp4Linear(v),
        lambda: Fp4Linear(w, v), lambda: Fp4FeedForward(lin, lin), lambda: Fp4FeedForward(lin, Fp4Linear(t, None), activation="x"),
        lambda: fp4_tensor_scale(torch.full((2, 2), math.inf)), lambda: Fp4Tensor.from_stored(t.codes, t.scales, 64, "nvfp4"),
        lambda: t.dequantize(torch.int8), lambda: t.dequantize(out=r),
    ):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K,offset", [(1, 40, 5120, 0), (1, 5000, 1000, 0), (2, 200, 320, 8), (5, 384, 1037, 1), (8, 130, 16, 0),
                                          (9, 24, 7, 3), (16, 1024, 2064, 0), (17, 256, 512, 0)])
def test_layer_of_few_rows(fmt, dtype, M, N, K, offset):
    """Quantised inside the product or in front of it: the same bits.  Rows a few elements apart, aligned or not; with NaN, zeros and
    infinity in single blocks."""
    g = gen(M + K)
    x = torch.randn(M, K + offset, generator=g).to(dtype).to(DEV)[:, offset:]
    if M > 2:
        x[1, :] = 0
        x[2, K // 2] = float("nan")
        x[2, K - 1] = float("inf")
    up = Fp4Linear((torch.randn(N, K, generator=g) / K ** 0.5).to(DEV), torch.randn(N, generator=g).to(dtype).to(DEV), fmt=fmt)
    down = Fp4Linear((torch.randn(72, N, generator=g) / N ** 0.5).to(DEV), fmt=fmt)
    a = fp4_quantize(x, fmt)
    want = fp4_matmul(a, up.w, bias=up.b, activation="silu", dtype=dtype)
    got = up(x, activation="silu")
    assert got.dtype == dtype and torch.equal(got.view(-1).view(torch.uint8), want.view(-1).view(torch.uint8))
    assert M <= 2 or bool(got[2].isnan().all()) and not bool(got[:2].isnan().any())
    want = fp4_matmul(fp4_matmul(a, up.w, bias=up.b, activation="gelu_tanh", dtype=fmt), down.w, dtype=dtype)
    assert torch.equal(Fp4FeedForward(up, down)(x).view(-1).view(torch.uint8), want.view(-1).view(torch.uint8))
    check_status()


@pytest.mark.parametrize("M", [1, 16])
def test_layer_of_few_rows_in_place(M):
    """Where the result overlaps the input, the input is read first."""
    g = gen(M)
    layer = Fp4Linear((torch.randn(2048, 2048, generator=g) / 45).to(BF).to(DEV))
    x = torch.randn(M, 2048, generator=g).to(BF).to(DEV)
    want = layer(x)
    for _ in range(20):
        y = x.clone()
        assert layer(y, out=y) is y and torch.equal(y, want)
    both = torch.zeros(M, 2048 + 8, dtype=BF, device=DEV)      # eight columns further on
    both[:, :2048] = x
    layer(both[:, :2048], out=both[:, 8:])
    assert torch.equal(both[:, 8:], want)
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M,K", [(1, 1536), (2, 6144), (1999, 1536), (1501, 6400), (900, 16384), (31, 16416)])
def test_modulated_rows_apart(fmt, M, K):
    """A row's codes do not depend on the rows that are quantised with it: each one alone gives the same bits, also next to one with a
    NaN."""
    g = gen(M + K)
    x = (torch.randn(M, K, generator=g) * 2 + 1).to(BF).to(DEV)
    if M > 1:
        x[M // 2, K // 3] = math.nan
    shift, scale = ((0.2 * torch.randn(K, generator=g)).to(BF).to(DEV) for _ in range(2))
    t = fp4_quantize(x, fmt, shift=shift, scale=scale)
    codes, s = t.to_stored()
    for m in {0, max(M // 2 - 1, 0), M // 2, min(M // 2 + 1, M - 1), M - 1}:
        one, s1 = fp4_quantize(x[m:m + 1], fmt, shift=shift, scale=scale).to_stored()
        assert torch.equal(one[0], codes[m]) and torch.equal(s1[0], s[m])
    bad = t.dequantize(F32).isnan().any(1)
    assert int(bad.sum()) == (M > 1) and (M == 1 or bool(bad[M // 2]))


@pytest.mark.parametrize("M", [1, 4, 16, 100, 700])
def test_chain_of_layers(M):
    """Every layer reads what the one before wrote, its workspace is the last one's memory: the same bits whether the host waits in
    between, does not, or replays a graph."""
    g = gen(M)
    layers = [Fp4Linear((torch.randn(512, 512, generator=g) / 22).to(BF).to(DEV), fmt=FMTS[i % 2]) for i in range(6)]
    x = torch.randn(M, 512, generator=g).to(BF).to(DEV)

    def chain(y, wait=False):
        for i in range(48):
            z = layers[i % 6](y, activation="silu" if i % 5 == 0 else None)
            y = z if i % 7 else z + y      # another kernel in between
            if wait:
                torch.cuda.synchronize()
        return y

    want = chain(x, wait=True)
    assert bool(want.isfinite().all()) and float(want.abs().max()) > 0
    for _ in range(5):
        assert torch.equal(chain(x), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(x)
    for _ in range(3):
        got.zero_()
        graph.replay()
        assert torch.equal(got, want)
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("M,N,off", [(3, 264, 8), (140, 136, 3), (1500, 1672, 8), (1500, 1672, 3)])
def test_activations_of_the_largest_arguments(fmt, dtype, activation, M, N, off):
    """Arguments whose square passes the range of 32 bits, infinities and NaN, in both kernels' epilogues: what the formula gives.  All but
    the first 32 columns are finite, so the blocks behind them are too."""
    a, w = stored(M, 64, fmt, M), stored(N, 64, fmt, N)
    a.tensor_scale = 2.0 ** -7
    large = torch.tensor([1e20, -1e20, 3e38, -3e38, 2e19, -2e19, 1.8e19, -1.8e19, 5.0, -5.0, 0.0, 1e30, -1e30, 1e10, -1e10, -80.0, 90.0])
    bias = large[torch.arange(N) % len(large)]
    bias[:4] = torch.tensor([math.inf, -math.inf, math.nan, 1e20])
    wide = torch.empty(M, N + 16, dtype=dtype, device=DEV)
    kw = dict(bias=bias.to(DEV), activation=activation)
    got = fp4_matmul(a, w, out=wide[:, off:off + N], **kw).cpu().double()
    want, size = plain64.matmul(values(a), values(w), bias=bias, activation=activation)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert bool((got[:, 0] == math.inf).all()) and bool(want[:, 3:].isfinite().all())
    err = (got - want).abs()[:, 3:]
    assert bool((err <= ULP[dtype] * want[:, 3:].abs() + 80 * 2.0 ** -23 * size[:, 3:]).all())
    quantised = fp4_matmul(a, w, dtype=fmt, **kw)
    for x, y in zip(codes_of(quantised), codes_of(fp4_quantize(fp4_matmul(a, w, dtype=F32, **kw), fmt))):
        assert torch.equal(x, y)
    assert bool(values(quantised)[:, 32:].isfinite().all())
    check_status()


@pytest.mark.parametrize("stuck,M,N,K", [(1, 1, 512, 2048), (1, 16, 40, 96), (1, 1500, 1672, 96), (1, 1500, 1672, 2080),
                                         (2, 1500, 1672, 96), (2, 3000, 5120, 96)])
def test_product_that_gave_up_says_so(lib, stuck, M, N, K):
    """Bytes that never come, of the first operands or of the last residuals: the waits run out, every CTA ends, the status says so, and the
    next product is as before.  Run with nothing missing in between."""
    a, w = stored(M, K, "nvfp4", 1), stored(N, K, "nvfp4", 2)
    residual = torch.randn(M, N, generator=gen(3)).to(BF).to(DEV)
    want = fp4_matmul(a, w, residual=residual)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.empty_like(want)

    def run(stuck):
        status.zero_()
        out.copy_(residual).mul_(0).sub_(7)
        code = lib.t2t_fp4_give_up_selftest(stuck, *a.pointers(), *w.pointers(), M, N, K, residual.data_ptr(), out.data_ptr(),
                                            status.data_ptr(), torch.cuda.current_stream().cuda_stream)
        assert code == 0
        return int(status.item())

    for _ in range(3):
        assert run(0) == 0 and torch.equal(out, want)
        assert run(stuck) == 1
        same = out == want
        assert not bool(same.all())
        if stuck == 2:      # only what lies behind the last residuals is missing
            assert bool((same | (out == -7)).all()) and bool(same.any())
    assert torch.equal(fp4_matmul(a, w, residual=residual), want)
    check_status()


def test_status_of_an_earlier_product_is_raised_once():
    """A product that gave up writes to its device's word; whatever is called next says so, and works from then on."""
    from token2tile_b200.fp4 import _status_of
    x = torch.randn(5, 64, generator=gen(1)).to(BF).to(DEV)
    layer = Fp4Linear(torch.randn(32, 64, generator=gen(2)).to(BF).to(DEV))
    back = Fp4Linear(torch.randn(64, 32, generator=gen(3)).to(BF).to(DEV))
    a = fp4_quantize(x)
    for call in (lambda: fp4_matmul(a, layer.w), lambda: fp4_matmul(a, layer.w, dtype="nvfp4"), lambda: layer(x), lambda: layer(x[:1]),
                 lambda: layer(a), lambda: Fp4FeedForward(layer, back)(x), check_status, lambda: check_status(wait=False)):
        call()
        _status_of(x.device).value.value = 1
        with pytest.raises(RuntimeError, match="fp4_matmul"):
            call()
        call()
    check_status()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("M", [3, 140, 1500])
def test_results_and_inputs_that_share_memory(fmt, M):
    """A factor is refused as the result; residuals some of whose elements the result overwrites are read first, by columns and by rows."""
    N = 1672 if M == 1500 else 264
    a, w, square = stored(M, 96, fmt, 1), stored(N, 96, fmt, 2), stored(N, N, fmt, 3)
    b = stored(M, N, fmt, 4)
    for factors, out in (((b, square), b), ((square, square), square)):
        with pytest.raises(ValueError, match="shares memory"):
            fp4_matmul(*factors, out=out)
    layer = Fp4Linear(w)
    x = torch.randn(M, 96, generator=gen(5)).to(BF).to(DEV)
    start = torch.randn(M + 3, N + 24, generator=gen(6)).to(BF).to(DEV)
    for rows, columns in ((0, 8), (0, 16), (1, 0), (2, 8), (-1, 0), (-3, -8), (0, -8)):
        r, c = max(-rows, 0), max(-columns, 0)
        residual = lambda t: t[r:r + M, c:c + N]
        result = lambda t: t[r + rows:r + rows + M, c + columns:c + columns + N]
        for call in (lambda **kw: fp4_matmul(a, w, **kw), lambda **kw: layer(x, **kw)):
            want = call(residual=residual(start).clone())
            buffer = start.clone()
            assert torch.equal(call(residual=residual(buffer), out=result(buffer)), want)
            result(buffer).copy_(result(start))
            assert torch.equal(buffer, start)
    check_status()


def test_refused_quantisation_leaves_its_output():
    x = torch.randn(3, 64, generator=gen(1)).to(DEV)
    for fmt, bad in (("nvfp4", (0.0, -1.0, math.nan, math.inf, 2.0 ** 101)), ("mxfp4", (2.0, 0.5))):
        t = fp4_quantize(x, fmt)
        want = t.dequantize()
        for g in bad:
            with pytest.raises(ValueError):
                fp4_quantize(x, fmt, tensor_scale=g, out=t)
            assert t.tensor_scale == 1.0 and torch.equal(t.dequantize(), want)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,K", [(1, 16), (3, 48), (130, 256), (9, 1000), (33, 5120), (700, 1001), (5, 16384), (5, 20481), (2, 30001)])
def test_modulated_quantize_with_wide_vectors(fmt, dtype, M, K):
    """32-bit shift and scale with rows of any type: values of x's type give the bits that they give as x's type; others what
    the formula gives, as near as in test_modulated_quantize."""
    g = gen(M + K)
    x = (torch.randn(M, K, generator=g) * 3 + torch.randn(M, 1, generator=g)).to(dtype)
    shift, scale = ((0.2 * torch.randn(K, generator=g)).to(dtype).to(DEV) for _ in range(2))
    codes = lambda **kw: fp4_quantize(x.to(DEV), fmt, **kw).to_stored()
    for a, b in zip(codes(shift=shift, scale=scale), codes(shift=shift.float(), scale=scale.float())):
        assert torch.equal(a, b)
    weight = torch.rand(K, generator=g) * 0.015 + 0.005      # of a norm: 16 bits do not hold its distance from 1
    shift = 0.01 * torch.randn(K, generator=g)
    t = fp4_quantize(x.to(DEV), fmt, shift=shift.to(DEV), scale=(weight - 1).to(DEV))
    y = plain64.modulated(x.double(), shift.double(), weight.double() - 1)
    _, s, value = plain64.quantize(y, fmt)
    got = values(t)
    # these rows lie where nvfp4's scales are subnormal and the definition itself is off by more than a step
    step = (s.repeat_interleave(plain64.BLOCK[fmt], 1)[:, :K]) * 2 * 1.2
    assert bool(((got - y).abs() <= (value - y).abs() + step * (2 if fmt == "mxfp4" else 1) + 1e-30).all())
    # weight - 1 in 32 bits is off by 2^-25, 6e-6 of the weight at most: one value in some thousand next to a middle or a scale's
    assert float((got != value).double().mean()) < 5e-3 + 40.0 / (M * K) * (M * K < 40000)
    layer = Fp4Linear((torch.randn(40, K, generator=g) / K ** 0.5).to(DEV), fmt=fmt)
    both = dict(shift=shift.to(DEV), scale=(weight - 1).to(DEV))
    assert torch.equal(layer(x.to(DEV), **both), layer(t, dtype=dtype))
    back = Fp4Linear(torch.randn(8, 40, generator=g).to(DEV), fmt=fmt)
    assert torch.equal(Fp4FeedForward(layer, back)(x.to(DEV), **both),
                       fp4_matmul(fp4_matmul(t, layer.w, activation="gelu_tanh", dtype=fmt), back.w, dtype=dtype))
    for bad in (dict(shift=shift.to(DEV).to(F16), scale=(weight - 1).to(DEV)), dict(shift=shift.to(DEV).double(), scale=shift.to(DEV).double())):
        for call in (lambda: fp4_quantize(x.to(DEV), fmt, **bad), lambda: layer(x.to(DEV), **bad)):
            with pytest.raises(ValueError):
                call()
    check_status()


def test_writing_to_out_is_seen_by_autograd():
    x = torch.randn(5, 64, generator=gen(1)).to(DEV)
    up, down = (Fp4Linear(torch.randn(n, k, generator=gen(n)).to(DEV)) for n, k in ((96, 64), (64, 96)))
    square, a = Fp4Linear(torch.randn(64, 64, generator=gen(3)).to(DEV)), fp4_quantize(x)
    for call in (lambda y: square(x, out=y), lambda y: square(y, out=y), lambda y: Fp4FeedForward(up, down)(x, out=y),
                 lambda y: fp4_matmul(a, square.w, out=y), lambda y: a.dequantize(out=y)):
        y, w = torch.ones(5, 64, device=DEV), torch.ones(64, device=DEV, requires_grad=True)
        loss = (y * w).sum()      # saves y
        call(y)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    t = Fp4Tensor.empty(5, 64, "nvfp4", device=DEV)
    for call in (lambda: fp4_quantize(x, out=t), lambda: fp4_matmul(a, square.w, out=t)):
        before = t.data._version
        call()
        assert t.data._version > before
    with torch.inference_mode():
        y = x.clone()
        assert square(y, out=y) is y
    check_status()


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("M,N", [(3, 264), (140, 136), (1500, 1672), (1500, 1671)])
def test_residual_of_one_row_for_all(dtype, M, N):
    """Broadcast over the rows (stride 0), or rows that overlap: the same bits as written out."""
    a, w = stored(M, 96, "nvfp4", 1), stored(N, 96, "nvfp4", 2)
    row = torch.randn(1, N, generator=gen(3)).to(dtype).to(DEV)
    for residual in (row.expand(M, N), torch.randn(8 * M + N, generator=gen(4)).to(dtype).to(DEV).as_strided((M, N), (8, 1))):
        want = fp4_matmul(a, w, residual=residual.contiguous(), dtype=dtype)
        assert torch.equal(fp4_matmul(a, w, residual=residual, dtype=dtype), want)
        out = torch.empty_like(want)
        assert torch.equal(fp4_matmul(a, w, residual=residual, out=out), want)
    layer, x = Fp4Linear(w), torch.randn(M, 96, generator=gen(5)).to(dtype).to(DEV)
    assert torch.equal(layer(x, residual=row.expand(M, N)), layer(x, residual=row.repeat(M, 1)))
    check_status()


@pytest.mark.parametrize("M", [2, 300])
def test_largest_tensor_scales(M):
    """Zeros stay zeros under the largest product of tensor scales that is taken."""
    a, w = (Fp4Tensor.empty(rows, 64, "nvfp4", g, DEV) for rows, g in ((M, 2.0 ** 100), (40, 2.0 ** 27)))
    for t in (a, w):
        t.data.zero_()
    assert not bool(fp4_matmul(a, w, dtype=F32).any())
    w.tensor_scale = 2.0 ** 28
    with pytest.raises(ValueError, match="32 bits"):
        fp4_matmul(a, w, dtype=F32)
    check_status()


def test_one_column():
    """Its stride means nothing, in any of the calls."""
    column = torch.randn(5, 8, generator=gen(1)).to(DEV)[:, ::4][:, :1]
    assert column.stride() == (8, 4)
    t = fp4_quantize(column)
    check_quantized(t, column)
    out = torch.zeros(5, 8, device=DEV)
    assert torch.equal(t.dequantize(out=out[:, ::4][:, :1]), t.dequantize()) and not bool(out[:, 1:].any())
    a, w = stored(5, 64, "nvfp4", 1), stored(1, 64, "nvfp4", 2)
    want = fp4_matmul(a, w, residual=column, dtype=F32)
    assert torch.equal(fp4_matmul(a, w, residual=column, out=out[:, ::4][:, :1]), want)
    check_status()


def test_range_of_a_layer():
    """A layer's own quantisation of nvfp4 holds magnitudes of 0.006 to 2,688; other rows are given quantised with their scale.  The weight, 6
    on its diagonal, is quantised exactly."""
    layer = Fp4Linear((6 * torch.eye(64)).to(BF).to(DEV))
    assert torch.equal(layer.w.dequantize(), 6 * torch.eye(64, device=DEV))
    row = lambda v: torch.full((5, 64), v, dtype=F32, device=DEV)
    held = lambda x, **kw: layer(x, **kw) / 6
    assert not bool(held(row(0.0058)).any()) and bool((held(row(0.006)) > 0.005).all())
    assert torch.equal(held(row(5000.0)), held(row(2688.0))) and bool((held(row(2688.0)) == 2688.0).all())
    for v in (1e-6, 3e5):
        g = fp4_tensor_scale(row(v))
        got = held(fp4_quantize(row(v), tensor_scale=g), dtype=F32)
        assert bool(((got / v - 1).abs() < 0.07).all())      # a scale has three bits behind its first
    check_status()
