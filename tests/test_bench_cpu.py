"""Host parts of the benchmark."""
import math

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
