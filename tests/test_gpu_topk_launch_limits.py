"""The operators built on the k largest of a row over more workgroups than one launch takes (2^32 threads along a dimension of
its grid): every row is served.  The rows that are looked at are the first, the last, and those on both sides of 2^31 threads;
all values are whole numbers or come out of a single rounding, so the results are exact."""
import numpy as np
import pytest

from zigrad_amd import HipDevice
from zigrad_amd.device import F32, U64

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dev():
    """A context of its own, which gives its memory back at the end of the test."""
    d = HipDevice(0)
    yield d
    d.deinit()


def places(rows, rows_per_group):
    """First rows, last rows, and those around the middle of the threads that one launch can have."""
    middle = (1 << 31) // 256 * rows_per_group
    return sorted({0, 1, middle - 1, middle, 2 * middle - 1, 2 * middle, rows - 2, rows - 1})


def row(dev, buf, r, n):
    return dev.to_numpy(buf.sub(r * n, n))


def test_selection_of_short_rows(dev):
    rows, cols, k = (1 << 28) + 21, 17, 2
    x, values, indices = dev.mem_alloc(F32, rows * cols), dev.mem_alloc(F32, rows * k), dev.mem_alloc(U64, rows * k)
    dev.mem_fill(x, -1.0)
    dev.mem_fill(values, 9.0)
    at = places(rows, 16)
    for i, r in enumerate(at):
        dev.mem_fill(x.sub(r * cols + 3 + i, 1), 5.0)
    dev.dispatch("topk_fwd", x=x, values=values, indices=indices, rows=rows, cols=cols, k=k)
    for i, r in enumerate(at):
        assert row(dev, values, r, k).tolist() == [5.0, -1.0] and row(dev, indices, r, k).tolist() == [3 + i, 0], r
    for r in (2, rows - 3):
        assert row(dev, values, r, k).tolist() == [-1.0, -1.0] and row(dev, indices, r, k).tolist() == [0, 1], r


# cols, k, rows a workgroup of 256 threads has: the kernels for short rows, for a row a wave, for a row (or more) a workgroup
@pytest.mark.parametrize("cols,k,per_group", [(1, 1, 16), (2, 17, 4), (1025, 1, 1)])
def test_the_gradient_of_a_selection(dev, cols, k, per_group):
    rows = (1 << 24) * per_group + 3 * per_group + 1
    indices, y_g, x_g = dev.mem_alloc(U64, rows * k), dev.mem_alloc(F32, rows * k), dev.mem_alloc(F32, rows * cols)
    dev.mem_fill(indices, cols - 1)
    dev.mem_fill(y_g, 1.0)
    dev.mem_fill(x_g, 9.0)
    at = places(rows, per_group) + [2, rows - 3]
    for i, r in enumerate(at):
        dev.mem_fill(y_g.sub(r * k, 1), 2.0 + i)
    dev.dispatch("topk_bwd", indices=indices, y_g=y_g, x_g=x_g, rows=rows, cols=cols, k=k, accumulate=False)
    for i, r in enumerate(at):
        want = np.zeros(cols, np.float32)
        want[-1] = 2 + i + k - 1
        assert np.array_equal(row(dev, x_g, r, cols), want), r


@pytest.mark.parametrize("fused", [False, True])
def test_distillation_of_short_rows_with_many_entries(dev, fused):
    """Two classes with the same logit, the teacher's 17 equal entries all on the second: q = 1/17 each and p = 1/2, so a row's
    loss is log 2 - log 17 and its gradient w (1/2, -1/2); rows of weight 0 add nothing."""
    rows, cols, k = (1 << 26) + 13, 2, 17
    at = places(rows, 4)
    b = {n: dev.mem_alloc(F32, s) for n, s in (("logits", rows * cols), ("teacher", rows * k), ("weights", rows), ("stats", 2 * rows),
                                               ("row_loss", rows), ("loss", 1), ("grad", rows * cols))}
    b["indices"] = dev.mem_alloc(U64, rows * k)
    for name, value in (("logits", 3.0), ("teacher", 0.0), ("indices", 1), ("weights", 0.0), ("stats", 9.0), ("row_loss", 9.0), ("grad", 9.0)):
        dev.mem_fill(b[name], value)
    for r in at:
        dev.mem_fill(b["weights"].sub(r, 1), 0.5)
    size = dict(rows=rows, cols=cols, k=k, temperature=1.0)
    loss, row_loss, grad = b.pop("loss"), b.pop("row_loss"), b.pop("grad")
    if fused:
        dev.dispatch("distill_fwd_bwd", loss=loss, row_loss=row_loss, grad=grad, accumulate=False, **b, **size)
    else:
        dev.dispatch("distill_fwd", loss=loss, row_loss=row_loss, **b, **size)
        dev.dispatch("distill_bwd", grad=grad, accumulate=False, **b, **size)
    # the logarithms are off by two halves of a step of their values each, their difference by one more, 17 sums of q by 17 of
    # a gradient below 1/2 and its factors by 8
    near, want = 2.0**-24 * (3 * np.log(34) + 25), np.log(2 / 17)
    for r in at:
        assert abs(row(dev, row_loss, r, 1)[0] - want) <= near, r
        assert np.abs(row(dev, grad, r, 2) - [0.25, -0.25]).max() <= near, r
    for r in (2, rows - 3):
        assert row(dev, row_loss, r, 1)[0] == 0 and (row(dev, grad, r, 2) == 0).all(), r
    assert abs(dev.to_numpy(loss)[0] - len(at) / 2 * want) <= len(at) * near


def test_one_expert_of_a_billion_rows(dev):
    n = (1 << 30) + 70
    x, y = dev.mem_alloc(F32, n), dev.mem_alloc(F32, n)
    w, gw = dev.from_numpy(np.full(1, 3, np.float32)), dev.from_numpy(np.full(1, 9, np.float32))
    offsets = dev.from_numpy(np.array([0, n - 1], np.uint64))
    dev.mem_fill(x, 0.0)
    dev.mem_fill(y, 9.0)
    at = [r for r in places(n, 64) if r < n - 1]
    for i, r in enumerate(at):
        dev.mem_fill(x.sub(r, 1), 1.0 + i)
    layer = dict(offsets=offsets, n_rows=n, n_experts=1, fan_in=1, fan_out=1)
    dev.dispatch("expert_linear_fwd", x=x, w=w, bias=None, y=y, relu=False, **layer)
    for i, r in enumerate(at):
        assert row(dev, y, r, 1)[0] == 3 * (1 + i), r
    assert row(dev, y, 2, 1)[0] == 0 and row(dev, y, n - 3, 1)[0] == 0 and row(dev, y, n - 1, 1)[0] == 9
    dev.mem_fill(y, 9.0)
    dev.dispatch("expert_linear_bwd", gy=x, x=x, w=w, act_in=None, gw=gw, gb=None, gx=y, accumulate=False, **layer)
    for i, r in enumerate(at):
        assert row(dev, y, r, 1)[0] == 3 * (1 + i), r
    assert row(dev, y, 2, 1)[0] == 0 and row(dev, y, n - 1, 1)[0] == 9
    assert dev.to_numpy(gw)[0] == sum((1 + i) ** 2 for i in range(len(at)))


@pytest.mark.parametrize("way", ["forward", "input gradient"])
def test_few_rows_of_very_wide_experts(dev, way):
    """A row for each of 256 experts with 2^21 - 1 outputs (or inputs): 16 columns a workgroup, tiles of every expert."""
    e, wide = 256, (1 << 21) - 1
    w, out = dev.mem_alloc(F32, e * wide), dev.mem_alloc(F32, e * wide)
    dev.mem_fill(w, 2.0)
    dev.mem_fill(out, 9.0)
    offsets = dev.from_numpy(np.arange(e + 1, dtype=np.uint64))
    narrow = dev.from_numpy(np.arange(1, e + 1, dtype=np.float32))
    if way == "forward":
        dev.dispatch("expert_linear_fwd", x=narrow, w=w, bias=None, y=out, relu=False, offsets=offsets, n_rows=e, n_experts=e, fan_in=1,
                     fan_out=wide)
    else:
        x, gw = dev.mem_alloc(F32, e * wide), dev.mem_alloc(F32, e * wide)
        dev.mem_fill(x, 1.0)
        dev.dispatch("expert_linear_bwd", gy=narrow, x=x, w=w, act_in=None, gw=gw, gb=None, gx=out, offsets=offsets, n_rows=e, n_experts=e,
                     fan_in=wide, fan_out=1, accumulate=False)
        assert (row(dev, gw, e - 1, wide) == e).all()
    for r in (0, 1, 62, 63, 64, 65, 127, 128, 129, e - 2, e - 1):
        assert (row(dev, out, r, wide) == 2 * (r + 1)).all(), r
