"""Offsets whose ranges overlap: outside the calls' contract for the rows' results, but nothing outside the ranges is touched and every
expert's weight and bias gradients are sums over its own range."""
import numpy as np
import pytest

from test_gpu_expert_linear import case, get, put

pytestmark = pytest.mark.gpu

# [offsets], rows that belong to no range.  Each with a range that ends before it begins between two that overlap.
OFFSETS = [([0, 60, 10, 60], []), ([0, 50, 0, 60], []), ([5, 30, 3, 59], [0, 1, 2, 59]), ([0, 60, 0, 60, 0, 60, 0, 60, 0, 60], []),
           ([0, 2**63, 7, 9], []), ([10, 20, 5, 15, 2, 12], [0, 1] + list(range(20, 60)))]


@pytest.mark.parametrize("offsets,free", OFFSETS)
@pytest.mark.parametrize("repeat", [1, 40])
@pytest.mark.parametrize("fan_in,fan_out", [(20, 24), (130, 68)])
def test_overlapping_ranges_stay_inside_themselves(hip, offsets, free, repeat, fan_in, fan_out):
    """repeat: each row stands for so many, which takes the tiled kernels.  Whole numbers: sums are exact in any order."""
    n, e = 60 * repeat, len(offsets) - 1
    c = case(1, [n] + [0] * (e - 1), 0, fan_in, fan_out)
    r = np.random.default_rng(n + e)
    for name in ("x", "w", "gy"):
        c[name] = r.integers(-4, 5, c[name].shape).astype(np.float32)
    ends = np.array([min(o * repeat, 2**64 - 1) for o in offsets], np.uint64)
    off = hip.from_numpy(ends)
    untouched = (np.array(free, int)[:, None] * repeat + np.arange(repeat)).ravel()
    b = {"x": put(hip, c["x"], 1), "w": put(hip, c["w"], 1), "gy": put(hip, c["gy"], 1), "y": put(hip, np.full((n, fan_out), 9, np.float32), 1),
         "gx": put(hip, np.full((n, fan_in), 9, np.float32), 1), "gw": put(hip, np.zeros(c["w"].shape, np.float32), 1),
         "gb": put(hip, np.zeros((e, fan_out), np.float32), 1)}
    layer = dict(offsets=off, n_rows=n, n_experts=e, fan_in=fan_in, fan_out=fan_out)
    hip.dispatch("expert_linear_fwd", x=b["x"][1], w=b["w"][1], bias=None, y=b["y"][1], relu=False, **layer)
    hip.dispatch("expert_linear_bwd", gy=b["gy"][1], x=b["x"][1], w=b["w"][1], act_in=None, gw=b["gw"][1], gb=b["gb"][1], gx=b["gx"][1],
                 accumulate=False, **layer)
    for name, shape in (("y", (n, fan_out)), ("gx", (n, fan_in))):
        assert (get(hip, b[name][0], 1, shape)[untouched] == 9).all(), name
    gw, gb = get(hip, b["gw"][0], 1, c["w"].shape), get(hip, b["gb"][0], 1, (e, fan_out))
    for k in range(e):
        rows = slice(min(int(ends[k]), n), min(int(ends[k + 1]), n))
        assert np.array_equal(gw[k], c["gy"][rows].T @ c["x"][rows]), k
        assert np.array_equal(gb[k], c["gy"][rows].sum(axis=0)), k
    for buf, _ in b.values():
        hip.mem_free(buf)
    hip.mem_free(off)
