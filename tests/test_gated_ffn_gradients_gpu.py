"""The block's gradients against central differences of its 64-bit definition, along the gradients themselves: there the slope is the
gradient's length and grows as the element-wise bounds do (1 to 7 % of it at these sizes), so a gradient that is missing, turned
round or a tenth off is beyond the bound, and the test says so of each.

Bound: what the element-wise tolerances allow along the direction, and 1e-6 of the slope for the difference itself (step 1e-4,
test_gated_ffn_gradients_cpu.py)."""
import pytest
import torch
from test_gated_ffn_gpu import BF, H, make, reference
from test_gated_ffn_gradients_cpu import slope_along

from sirius_b200 import ops

pytestmark = pytest.mark.gpu


# a few tokens, one tile not filled, outputs of single CTAs through shared memory, pairs of CTAs
@pytest.mark.parametrize("t,c,f", [(3, 72, 40), (70, 136, 264), (300, 264, 520), (1100, 136, 264)])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_along_the_gradients(t, c, f, dtype):
    s = make(t, c, f)
    got = ops.gated_ffn_backward(s["dy"], s["x"], s["wgu"], s["wd"], grad_dtype=dtype)
    assert ops.tc_status() == 0
    base = [s["x"].double(), s["wgu"].double(), s["wd"].double()]
    _, tol = reference(s["x"], s["wgu"], s["wd"], dy=s["dy"])
    parts = [(0, slice(None)), (1, slice(0, f)), (1, slice(f, 2 * f)), (2, slice(None))]   # gate and up each by itself
    for k, rows in parts:
        g = got[k].double()
        d = torch.zeros_like(g)
        d[rows] = g[rows] / g[rows].norm()
        slope = slope_along(base, s["dy"].double(), k, d)
        rounded = H if k == 0 or dtype == BF else 2.0 ** -23
        bound = float(((tol[k] + rounded * (g.abs() + tol[k])) * d.abs()).sum()) * 1.01 + 1e-6 * abs(slope)
        agrees = lambda grad: abs(float((grad * d).sum()) - slope) <= bound
        assert agrees(g), (k, rows)
        for wrong in (torch.zeros_like(g), -g, 1.1 * g, 0.9 * g):
            assert not agrees(wrong), (k, rows, bound, slope)
