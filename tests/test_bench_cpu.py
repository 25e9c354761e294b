"""Host parts of the benchmark."""
import math
import types

import pytest

import bench


def test_roofline_of_the_transformer_step():
    """4-bit products stand against the 4-bit rate, four times the bf16 one."""
    pk = dict(tf=1400.0, src="measured")
    bf = bench.dit_roofline(None, 700e12, 1000.0, pk)
    assert bf["peak"] == 1400.0 and math.isclose(bf["achieved"], 700.0) and math.isclose(bf["frac"], 0.5) and "4 x" not in bf["note"]
    for fmt in ("nvfp4", "mxfp4"):
        r = bench.dit_roofline(fmt, 700e12, 1000.0, pk)
        assert r["peak"] == 5600.0 and math.isclose(r["achieved"], 700.0) and math.isclose(r["frac"], 0.125)
        assert fmt in r["kernel"] and "derived" in r["note"]


def test_waits_that_gave_up_end_the_measurement(monkeypatch):
    """Those of the attention, and those of 4-bit products whatever the attention is."""
    from token2tile_b200 import fp4
    asked = []

    def gave_up(dev):
        asked.append(dev)
        raise RuntimeError("wait timed out")

    monkeypatch.setattr(fp4, "check_status", gave_up)
    runtime = lambda code: types.SimpleNamespace(deploy=types.SimpleNamespace(device_status=lambda: code))
    bench.check_waits("cuda:0", None, [runtime(0)])
    with pytest.raises(AssertionError):
        bench.check_waits("cuda:0", None, [runtime(0), runtime(1)])
    assert not asked
    for runtimes in ([], [runtime(0)]):
        with pytest.raises(RuntimeError):
            bench.check_waits("cuda:0", "nvfp4", runtimes)
    assert asked == ["cuda:0"] * 2
    assert bench.dit_measure.__code__.co_names.count("check_waits") == 1
