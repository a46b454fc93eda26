"""Selection and distillation over the longest rows there are, 2^31 - 1 columns (8.6 GB each): a row that falls from its first column on,
with its largest values planted near the end, in the middle and at the start."""
import numpy as np
import pytest

from topk_reference import distill, distill_bounds
from zigrad_amd import HipDevice
from zigrad_amd.device import F32, U64

pytestmark = pytest.mark.gpu
COLS = (1 << 31) - 1
PLANTED = {COLS - 1: 9.0, COLS - 2: 3.0, COLS - 4096: 8.0, (1 << 30) + 5: 7.0, 1 << 30: 6.0, 70_000: 5.0, 3: 4.0}


@pytest.fixture(scope="module")
def row():
    """A context of its own (the memory goes back at the end) and the row; the columns from 300 on are below -299."""
    d = HipDevice(0)
    x = d.mem_alloc(F32, COLS)
    d.mem_sequence(x, 0.0, -1.0)
    for c, v in PLANTED.items():
        d.mem_fill(x.sub(c, 1), v)
    yield d, x
    d.deinit()


def largest(k):
    order = sorted(PLANTED, key=lambda c: -PLANTED[c]) + [c for c in range(k + 8) if c not in PLANTED]
    values = [PLANTED.get(c, -float(c)) for c in order]
    return np.array(order[:k], np.uint64), np.array(values[:k], np.float32)


@pytest.mark.parametrize("k", [1, 5, 100, 200, 512])
def test_selection_and_its_gradient(row, k):
    d, x = row
    values, indices, x_g = d.mem_alloc(F32, k), d.mem_alloc(U64, k), d.mem_alloc(F32, COLS)
    d.dispatch("topk_fwd", x=x, values=values, indices=indices, rows=1, cols=COLS, k=k)
    want_i, want_v = largest(k)
    assert np.array_equal(d.to_numpy(indices), want_i) and np.array_equal(d.to_numpy(values), want_v)
    d.mem_fill(x_g, 2.0)
    for accumulate in (True, False):
        d.dispatch("topk_bwd", indices=indices, y_g=values, x_g=x_g, rows=1, cols=COLS, k=k, accumulate=accumulate)
        base = 2.0 if accumulate else 0.0
        for c, v in zip(want_i[:8], want_v[:8]):
            assert d.to_numpy(x_g.sub(int(c), 1))[0] == base + v
        assert d.to_numpy(x_g.sub(COLS - 3, 1))[0] == base and d.to_numpy(x_g.sub((1 << 30) + 1, 4)).tolist() == [base] * 4
    for b in (values, indices, x_g):
        d.mem_free(b)


@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_distillation(row, fused, add):
    """The same loss over the planted columns and the first 300 alone: e^-299 adds nothing to a sum of 64 bits."""
    d, x = row
    k = 6
    at, _ = largest(7)
    at = at[[0, 1, 2, 3, 4, 6]]
    teacher = np.array([[3.0, 2.0, 1.5, 1.0, 0.5, 0.0]], np.float32)
    b = {"teacher": d.from_numpy(teacher), "indices": d.from_numpy(at), "stats": d.mem_alloc(F32, 2), "row_loss": d.mem_alloc(F32, 1),
         "loss": d.mem_alloc(F32, 1), "grad": d.mem_alloc(F32, COLS)}
    d.mem_fill(b["grad"], 0.25)
    loss = dict(logits=x, teacher=b["teacher"], indices=b["indices"], stats=b["stats"], rows=1, cols=COLS, k=k, temperature=1.0)
    if fused:
        d.dispatch("distill_fwd_bwd", row_loss=b["row_loss"], loss=b["loss"], grad=b["grad"], accumulate=add, **loss)
    else:
        d.dispatch("distill_fwd", row_loss=b["row_loss"], loss=b["loss"], **loss)
        d.dispatch("distill_bwd", grad=b["grad"], accumulate=add, **loss)
    seen = sorted(set(range(300)) | set(PLANTED))
    short = np.array([[PLANTED.get(c, -float(c)) for c in seen]], np.float32)
    where = {c: i for i, c in enumerate(seen)}
    ref = distill(short, teacher, np.array([[where[int(c)] for c in at]], np.uint64), 1.0)
    tol = distill_bounds(ref, short, 1.0, np.ones(1))
    got = d.to_numpy(b["stats"])
    assert got[0] == 9.0 and abs(got[1] - ref["stats"][0, 1]) <= tol["ls"][0]
    assert abs(d.to_numpy(b["row_loss"])[0] - ref["row_loss"][0]) <= tol["row_loss"][0]
    assert abs(d.to_numpy(b["loss"])[0] - ref["loss"]) <= tol["row_loss"][0]
    base = 0.25 if add else 0.0
    for c in seen:
        want, g = base + ref["grad"][0, where[c]], d.to_numpy(b["grad"].sub(c, 1))[0]
        assert abs(g - want) <= tol["grad"][0, where[c]] + 2.0**-24 * 2 * abs(want) * add + 2.0**-126, c
    for c in (400, 1 << 29, (1 << 30) + 4, COLS - 3):
        assert d.to_numpy(b["grad"].sub(c, 1))[0] == base, c
    for buf in b.values():
        d.mem_free(buf)
