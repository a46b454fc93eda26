"""The operators built on the k largest of a row on matrices of more than 2^32 elements, and the products of layers whose weights
pass 2^32: the places that are looked at lie behind the 32-bit mark."""
import numpy as np
import pytest

from topk_reference import distill, distill_bounds, topk
from zigrad_amd.device import F32, U64

pytestmark = pytest.mark.gpu
COLS = 40_000
ROWS = (1 << 32) // COLS + 3  # 107377 rows, 17 GB


def test_selection_and_distillation(hip):
    r = np.random.default_rng(1)
    last = r.standard_normal((2, COLS)).astype(np.float32)
    x, k = hip.mem_alloc(F32, ROWS * COLS), 64
    values, indices = hip.mem_alloc(F32, ROWS * k), hip.mem_alloc(U64, ROWS * k)
    grad = hip.mem_alloc(F32, ROWS * COLS)
    stats, row_loss, loss = hip.mem_alloc(F32, 2 * ROWS), hip.mem_alloc(F32, ROWS), hip.mem_alloc(F32, 1)
    w = np.zeros(ROWS, np.float32)
    w[-2:] = 0.5
    weights = hip.from_numpy(w)
    try:
        hip.mem_fill(x, -3.0)
        hip.mem_transfer(last, x.sub((ROWS - 2) * COLS, 2 * COLS), "HtoD")
        hip.dispatch("topk_fwd", x=x, values=values, indices=indices, rows=ROWS, cols=COLS, k=k)
        want_v, want_i = topk(last, k)
        assert np.array_equal(hip.to_numpy(indices.sub((ROWS - 2) * k, 2 * k), (2, k)), want_i)
        assert np.array_equal(hip.to_numpy(values.sub((ROWS - 2) * k, 2 * k), (2, k)), want_v)
        assert np.array_equal(hip.to_numpy(indices.sub(0, k)), np.arange(k, dtype=np.uint64))  # equal values: by column
        # the student's own best as teacher, one temperature up: its rows alone count
        ref = distill(last, want_v, want_i, 2.0, w[-2:])
        tol = distill_bounds(ref, last, 2.0, w[-2:].astype(np.float64))
        for fused in (True, False):
            hip.mem_fill(grad, 7.0)
            p = dict(logits=x, teacher=values, indices=indices, weights=weights, stats=stats, rows=ROWS, cols=COLS, k=k, temperature=2.0)
            if fused:
                hip.dispatch("distill_fwd_bwd", row_loss=row_loss, loss=loss, grad=grad, accumulate=False, **p)
            else:
                hip.dispatch("distill_fwd", row_loss=row_loss, loss=loss, **p)
                hip.dispatch("distill_bwd", grad=grad, accumulate=False, **p)
            got = hip.to_numpy(grad.sub((ROWS - 2) * COLS, 2 * COLS), (2, COLS))
            assert (np.abs(got - ref["grad"]) <= tol["grad"] + 2.0**-126).all()
            assert (np.abs(hip.to_numpy(row_loss.sub(ROWS - 2, 2)) - ref["row_loss"]) <= tol["row_loss"]).all()
            assert (hip.to_numpy(grad.sub(COLS, COLS)) == 0).all() and (hip.to_numpy(grad.sub((ROWS - 3) * COLS, COLS)) == 0).all()
        y_g = values
        hip.dispatch("topk_bwd", indices=indices, y_g=y_g, x_g=grad, rows=ROWS, cols=COLS, k=k, accumulate=False)
        want = np.zeros((2, COLS), np.float32)
        np.put_along_axis(want, want_i.astype(np.int64), want_v, axis=1)
        assert np.array_equal(hip.to_numpy(grad.sub((ROWS - 2) * COLS, 2 * COLS), (2, COLS)), want)
        hip.dispatch("topk_bwd", indices=indices, y_g=y_g, x_g=grad, rows=ROWS, cols=COLS, k=k, accumulate=True)
        assert np.array_equal(hip.to_numpy(grad.sub((ROWS - 2) * COLS, 2 * COLS), (2, COLS)), want + want)
    finally:
        for b in (x, values, indices, grad, stats, row_loss, loss, weights):
            hip.mem_free(b)


def test_rows_to_experts_and_back(hip):
    """2^19 + 5 tokens, two entries each, rows of 4100 values: 4.3e9 values in the experts' order."""
    tokens, k, width, n_experts = (1 << 19) + 5, 2, 4100, 16
    n = tokens * k
    r = np.random.default_rng(2)
    experts = r.integers(0, n_experts, n).astype(np.uint64)
    experts[-2:] = n_experts - 1  # the last token's rows are the last ones
    marks = r.integers(-8, 9, (1, width)).astype(np.float32)
    e, offsets, slots = hip.from_numpy(experts), hip.mem_alloc(U64, n_experts + 1), hip.mem_alloc(U64, n)
    x, y, out = hip.mem_alloc(F32, tokens * width), hip.mem_alloc(F32, n * width), hip.mem_alloc(F32, tokens * width)
    w, w_g = hip.mem_alloc(F32, n), hip.mem_alloc(F32, n)
    try:
        assert n * width > 1 << 32
        hip.mem_fill(x, 1.0)
        hip.mem_fill(w, 0.5)
        hip.mem_transfer(marks, x.sub((tokens - 1) * width, width), "HtoD")
        hip.dispatch("expert_sort", experts=e, offsets=offsets, slots=slots, n_experts=n_experts)
        assert hip.to_numpy(slots.sub(n - 1, 1))[0] == n - 1
        size = dict(n_tokens=tokens, k=k, width=width)
        hip.dispatch("expert_dispatch", x=x, slots=slots, y=y, **size)
        assert np.array_equal(hip.to_numpy(y.sub((n - 1) * width, width)), marks[0])
        hip.dispatch("expert_combine", y=y, slots=slots, weights=w, out=out, **size)
        assert np.array_equal(hip.to_numpy(out.sub((tokens - 1) * width, width)), marks[0])   # a half twice
        hip.dispatch("expert_dispatch_bwd", y_g=y, slots=slots, x_g=out, accumulate=True, **size)
        assert np.array_equal(hip.to_numpy(out.sub((tokens - 1) * width, width)), 3 * marks[0])
        hip.dispatch("expert_combine_bwd", out_g=out, y=y, slots=slots, weights=w, y_g=None, weights_g=w_g, **size)
        assert hip.to_numpy(w_g.sub(n - 1, 1))[0] == 3 * (marks[0].astype(np.float64) ** 2).sum()   # whole numbers below 2^24
        hip.dispatch("expert_combine_bwd", out_g=out, slots=slots, weights=w, y_g=y, **size)
        assert np.array_equal(hip.to_numpy(y.sub((n - 1) * width, width)), 1.5 * marks[0])
    finally:
        for b in (e, offsets, slots, x, y, out, w, w_g):
            hip.mem_free(b)


@pytest.mark.parametrize("per", [3, 40])
def test_layers_of_experts(hip, per):
    """1024 experts of 2050 x 2056: 4.3e9 weights; the last expert's products, through the kernels for few rows and the tiled ones."""
    n_experts, fan_in, fan_out = 1024, 2056, 2050
    r = np.random.default_rng(per)
    counts = np.full(n_experts, per)
    counts[::2] = 0
    counts[-1] = per
    n = int(counts.sum())
    offsets = hip.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.uint64))
    x, gy = r.integers(-4, 5, (n, fan_in)).astype(np.float32), r.integers(-4, 5, (n, fan_out)).astype(np.float32)
    w_last = r.integers(-4, 5, (fan_out, fan_in)).astype(np.float32)
    size = n_experts * fan_in * fan_out
    assert size > 1 << 32
    b = {"x": hip.from_numpy(x), "gy": hip.from_numpy(gy), "w": hip.mem_alloc(F32, size), "gw": hip.mem_alloc(F32, size),
         "y": hip.mem_alloc(F32, n * fan_out), "gx": hip.mem_alloc(F32, n * fan_in)}
    try:
        hip.mem_fill(b["w"], 0.0)
        hip.mem_fill(b["gw"], 1.0)
        hip.mem_transfer(w_last, b["w"].sub(size - fan_in * fan_out, fan_in * fan_out), "HtoD")
        layer = dict(offsets=offsets, n_rows=n, n_experts=n_experts, fan_in=fan_in, fan_out=fan_out)
        hip.dispatch("expert_linear_fwd", x=b["x"], w=b["w"], bias=None, y=b["y"], relu=False, **layer)
        hip.dispatch("expert_linear_bwd", gy=b["gy"], x=b["x"], w=b["w"], act_in=None, gw=b["gw"], gb=None, gx=b["gx"], accumulate=True,
                     **layer)
        # whole numbers below 2^24: exact in any order
        y, gx = hip.to_numpy(b["y"], (n, fan_out)), hip.to_numpy(b["gx"], (n, fan_in))
        assert np.array_equal(y[-per:], x[-per:] @ w_last.T) and (y[:-per] == 0).all()
        assert np.array_equal(gx[-per:], gy[-per:] @ w_last) and (gx[:-per] == 0).all()
        gw = hip.to_numpy(b["gw"].sub(size - fan_in * fan_out, fan_in * fan_out), (fan_out, fan_in))
        assert np.array_equal(gw, 1 + gy[-per:].T @ x[-per:])
        assert (hip.to_numpy(b["gw"].sub(size - 2 * fan_in * fan_out, fan_in * fan_out)) == 1).all()
    finally:
        for buf in (*b.values(), offsets):
            hip.mem_free(buf)
