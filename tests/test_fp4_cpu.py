"""4-bit floating point without a GPU: sizes, refusals of the C entries, and the 64-bit definition against hand-made values."""
import math
import pathlib

import torch

import plain64
from token2tile_b200.fp4 import FEW_ROWS, Fp4Tensor, fp4_tensor_scale


def test_sizes(lib):
    assert lib.t2t_fp4_codes_bytes(3, 33) == 3 * 32 and lib.t2t_fp4_codes_bytes(3, 32) == 3 * 16
    assert lib.t2t_fp4_scales_bytes(129, 64, 1) == 2 * 512 and lib.t2t_fp4_scales_bytes(128, 129, 0) == 2 * 512
    assert lib.t2t_fp4_codes_bytes(0, 5) == 0 and lib.t2t_fp4_scales_bytes(1, 1, 7) == 0
    for rows, K, fmt in ((1, 1, "mxfp4"), (300, 1000, "nvfp4"), (128, 128, "mxfp4")):
        t = Fp4Tensor.empty(rows, K, fmt, device="cpu")
        assert t.codes.numel() == lib.t2t_fp4_codes_bytes(rows, K)
        assert t.scales.numel() == lib.t2t_fp4_scales_bytes(rows, K, ("mxfp4", "nvfp4").index(fmt))


def test_entry_points_refuse_bad_arguments(lib):
    x = 4096                     # never read: every call is refused before anything is launched

    def quantize(p=x, stride=64, shift=0, scale=0, M=4, K=64, dtype=0, fmt=1, g=1.0, codes=x, scales=x):
        return lib.t2t_fp4_quantize(p, stride, shift, scale, 1e-6, M, K, dtype, fmt, g, codes, scales, 0)

    for kw in (dict(p=0), dict(codes=0), dict(scales=0), dict(codes=x + 8), dict(stride=-1), dict(shift=x), dict(scale=x), dict(M=0),
               dict(K=0), dict(K=1 << 25), dict(dtype=3), dict(fmt=2), dict(fmt=-1), dict(g=0.0), dict(g=math.inf), dict(g=math.nan),
               dict(g=-1.0), dict(fmt=0, g=2.0)):
        assert quantize(**kw) == 1, kw
    assert lib.t2t_fp4_dequantize(0, x, 4, 64, 1, 1.0, x, 64, 0, 0) == 1
    assert lib.t2t_fp4_dequantize(x, x, 4, 64, 1, 1.0, x, 63, 0, 0) == 1
    assert lib.t2t_fp4_dequantize(x, x, 4, 64, 1, 1.0, x, 64, 9, 0) == 1

    def matmul(a=x, w=x, M=4, N=8, K=64, fmt=1, act=0, vd=0, stride=8, out=x, dtype=0, res=0, rs=0):
        return lib.t2t_fp4_matmul(a, x, w, x, M, N, K, fmt, 1.0, 0, act, 0, vd, res, rs, out, stride, dtype, 0, 0)

    for kw in (dict(a=0), dict(w=0), dict(out=0), dict(M=0), dict(N=0), dict(K=0), dict(fmt=3), dict(act=3), dict(act=-1), dict(vd=3),
               dict(dtype=-1), dict(stride=7), dict(res=x, rs=-8)):
        assert matmul(**kw) == 1, kw


    def product(fmt=1, g=1.0, codes=x, scales=x):
        return lib.t2t_fp4_matmul_quantize(x, x, x, x, 4, 8, 64, fmt, 1.0, 0, 0, 0, 0, g, codes, scales, 0, 0)

    def linear(p=x, ws=x, size=1 << 20, fmt=1, M=4, shift=0, out=x):
        return lib.t2t_fp4_linear(p, 64, shift, 0, 1e-6, M, 64, 0, fmt, x, x, 1.0, 8, 0, 0, 0, 0, 0, 0, out, 8, ws, size, 0, 0)

    def ffn(p=x, ws=x, size=1 << 20, F=96, act=1):
        return lib.t2t_fp4_feed_forward(p, 64, 0, 0, 1e-6, 4, 64, 0, 1, x, x, 1.0, F, 0, 0, act, x, x, 1.0, 8, 0, 0, 0, 0, 0, x, 8, ws,
                                        size, 0, 0)

    for kw in (dict(p=0), dict(ws=0), dict(F=0)):
        assert ffn(**kw) == 1, kw
    assert ffn(size=lib.t2t_fp4_feed_forward_ws_bytes(4, 64, 96, 1) - 1) == 3
    for kw in (dict(p=0), dict(ws=0), dict(fmt=5), dict(M=0), dict(shift=x)):
        assert linear(**kw) == 1, kw
    assert linear(size=lib.t2t_fp4_linear_ws_bytes(4, 64, 1) - 1) == 3
    for kw in (dict(codes=0), dict(codes=x + 4), dict(scales=0), dict(g=0.0), dict(fmt=0, g=2.0), dict(fmt=2)):
        assert product(**kw) == 1, kw


def test_definition():
    x = torch.tensor([[6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.26, -0.74] + [0.0] * 6], dtype=torch.float64)
    code, scale, value = plain64.quantize(x, "nvfp4")
    assert scale.tolist() == [[1.0]] and code[0, :10].tolist() == [7, 0, 2, 2, 4, 4, 6, 6, 9, 9]
    code, scale, value = plain64.quantize(x * 1.3, "mxfp4")      # 7.8 saturates under the scale 1
    assert scale.tolist() == [[1.0]] and float(value[0, 0]) == 6.0
    assert plain64.quantize(torch.zeros(1, 32, dtype=torch.float64), "mxfp4")[1].tolist() == [[2.0 ** -127]]
    y = x.clone()
    y[0, 3] = math.nan
    assert bool(plain64.quantize(y, "nvfp4")[2].isnan().all())


def test_tensor_scale():
    assert fp4_tensor_scale(torch.tensor([2688.0])) == 1.0 and fp4_tensor_scale(torch.tensor([2689.0])) == 2.0
    assert fp4_tensor_scale(torch.zeros(3)) == 2.0 ** -100      # its lowest value


def test_few_rows():
    header = (pathlib.Path(__file__).parents[1] / "include" / "t2t_b200.h").read_text()
    assert f"#define T2T_FP4_FEW_ROWS {FEW_ROWS}\n" in header


def test_give_up_selftest_refuses_bad_arguments(lib):
    x = 4096                     # never read

    def call(stuck=1, a=x, M=4, N=8, K=64, residual=x, out=x, status=x):
        return lib.t2t_fp4_give_up_selftest(stuck, a, x, x, x, M, N, K, residual, out, status, 0)

    for kw in (dict(stuck=-1), dict(stuck=3), dict(a=0), dict(a=x + 8), dict(M=0), dict(N=0), dict(N=9), dict(K=0), dict(residual=0), dict(out=0),
               dict(out=x + 2), dict(status=0)):
        assert call(**kw) == 1, kw


def test_results_that_overlap_a_factor_are_refused(lib):
    """Other CTAs would still read what the first ones overwrite."""
    at = dict(a=1 << 20, a_scales=2 << 20, w=3 << 20, w_scales=4 << 20)      # never read
    M, N, K = 300, 64, 64
    codes, scales = lib.t2t_fp4_codes_bytes, lib.t2t_fp4_scales_bytes

    def quantised(out, out_scales):
        return lib.t2t_fp4_matmul_quantize(at["a"], at["a_scales"], at["w"], at["w_scales"], M, N, K, 1, 1.0, 0, 0, 0, 0, 1.0, out,
                                           out_scales, 0, 0)

    free = 8 << 20
    for name, size in (("a", codes(M, K)), ("a_scales", scales(M, K, 1)), ("w", codes(N, K)), ("w_scales", scales(N, K, 1))):
        for p in (at[name], at[name] + size - 16, at[name] - 16):
            assert quantised(p, free) == 1 and quantised(free, p) == 1, name
            assert lib.t2t_fp4_matmul(at["a"], at["a_scales"], at["w"], at["w_scales"], M, N, K, 1, 1.0, 0, 0, 0, 0, 0, 0, p, N, 0, 0,
                                      0) == 1, name


def test_residuals_that_the_result_overlaps_are_copied():
    """But not the result's own, nor other columns of one wide matrix, nor a row for all."""
    from token2tile_b200.fp4 import _beside
    wide = torch.arange(20 * 64, dtype=torch.float32).view(20, 64)
    out = wide[4:12, 16:32]
    for kept in (out, wide[4:12, :16], wide[4:12, 32:48], wide[:8, 40:56], wide[12:20, 16:32], wide[13:14, :16].expand(8, 16),
                 torch.zeros(8, 16), wide[11:19, :16], wide[5:13, :16]):
        assert _beside(kept, out) is kept
    for other in (wide[5:13, 16:32], wide[3:11, 16:32], wide[4:12, 17:33], wide[4:12, 1:17], wide[11:19, 1:17], wide[0:8, 31:47],
                  wide[6:7, 20:36].expand(8, 16), wide.view(-1)[4 * 64:][:128].view(8, 16)):
        got = _beside(other, out)
        assert got is not other and torch.equal(got, other) and got.untyped_storage().data_ptr() != wide.untyped_storage().data_ptr()
    one = wide[4:5]      # one row: the stride means nothing
    assert _beside(wide.view(10, 128)[2:3, :64], one) is not None and _beside(wide[4:5], one) is not None
    row = wide.view(10, 128)[2:3, :64]
    assert row.data_ptr() == one.data_ptr() and _beside(row, one) is row
    half = wide[4:5].clone()
    assert _beside(half, one) is half and _beside(wide.view(-1)[4 * 64 + 8:][:64].view(1, 64), one).data_ptr() != one.data_ptr() + 32


def test_wide_vectors(lib):
    from token2tile_b200.fp4 import WIDE_VECTORS
    header = (pathlib.Path(__file__).parents[1] / "include" / "t2t_b200.h").read_text()
    assert f"T2T_WIDE_VECTORS = {WIDE_VECTORS:#x} " in header
    x = 4096                     # never read
    for dtype in (3, WIDE_VECTORS + 3, WIDE_VECTORS * 2, -1):
        assert lib.t2t_fp4_quantize(x, 64, x, x, 1e-6, 4, 64, dtype, 1, 1.0, x, x, 0) == 1


def test_a_device_has_one_status_word(monkeypatch):
    """Threads whose first calls meet get the same word: kernels of both write to what either reads."""
    import threading
    import time
    import types

    from token2tile_b200 import fp4

    class Slow:
        def __init__(self):
            time.sleep(0.05)

    monkeypatch.setattr(fp4, "_Status", Slow)
    monkeypatch.setattr(fp4, "_status", {})
    start, got = threading.Barrier(8), []

    def ask(index):
        start.wait()
        got.append((index, fp4._status_of(types.SimpleNamespace(index=index))))

    threads = [threading.Thread(target=ask, args=(i % 2,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 8 and all(s is fp4._status[i] for i, s in got) and fp4._status[0] is not fp4._status[1]


def test_refuses_matrices_on_the_host():
    import pytest

    from token2tile_b200 import Fp4FeedForward, Fp4Linear, fp4_matmul
    a, w = Fp4Tensor.empty(3, 64, "nvfp4", device="cpu"), Fp4Tensor.empty(64, 64, "nvfp4", device="cpu")
    x, layer = torch.zeros(3, 64), Fp4Linear(w)
    for call in (a.dequantize, lambda: fp4_matmul(a, w), lambda: fp4_matmul(a, w, dtype="nvfp4"), lambda: layer(a), lambda: layer(x),
                 lambda: Fp4FeedForward(layer, layer)(x)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_tensor_scales_whose_product_has_no_32_bits(lib):
    import pytest

    from token2tile_b200 import fp4_matmul
    x = 4096                     # never read
    for alpha in (math.inf, -math.inf, math.nan):
        assert lib.t2t_fp4_matmul(x, 2 * x, 3 * x, 4 * x, 4, 8, 64, 1, alpha, 0, 0, 0, 0, 0, 0, 5 * x, 8, 0, 0, 0) == 1
    a, w = (Fp4Tensor.empty(3, 64, "nvfp4", g, device="cpu") for g in (2.0 ** 100, 2.0 ** 28))
    with pytest.raises(ValueError, match="32 bits"):
        fp4_matmul(a, w)
