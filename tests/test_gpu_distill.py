"""The loss against a teacher's k largest logits and its gradient against the formula in 64 bits, with bounds counted in
roundings (topk_reference.distill_bounds), and the formula against differences."""
import numpy as np
import pytest

from topk_reference import EPS, distill, distill_bounds

pytestmark = pytest.mark.gpu
U64 = np.uint64


def case(seed, rows, cols, k, scale=2.0):
    r = np.random.default_rng(seed)
    x = (r.standard_normal((rows, cols)) * scale).astype(np.float32)
    indices = ((r.integers(0, cols, (rows, 1)) + np.arange(k)) % cols).astype(U64)
    teacher = -np.sort(-(r.standard_normal((rows, k)) * scale).astype(np.float32), axis=1)
    return x, teacher, indices, (r.standard_normal((rows, cols)) / rows).astype(np.float32)


def run(hip, x, teacher, indices, temp, weights=None, grad0=None, fused=False, guard=16):
    """stats, row_loss, loss and gradient of the two calls, or of the fused one; grad0: the gradient to add to."""
    rows, cols = x.shape
    k = teacher.shape[1]
    b = {"logits": hip.from_numpy(x), "teacher": hip.from_numpy(teacher), "indices": hip.from_numpy(indices)}
    if weights is not None:
        b["weights"] = hip.from_numpy(weights)
    stats, row_loss, loss = (hip.from_numpy(np.full(n, 9.0, np.float32)) for n in (2 * rows, rows, 1))
    fill = np.full(x.size, 11.0, np.float32) if grad0 is None else grad0.ravel()
    g = hip.from_numpy(np.concatenate([np.full(guard, 3.5, np.float32), fill, np.full(guard, 3.5, np.float32)]))
    grad = g.sub(guard, x.size)
    size = dict(rows=rows, cols=cols, k=k, temperature=temp)
    if fused:
        hip.dispatch("distill_fwd_bwd", stats=stats, row_loss=row_loss, loss=loss, grad=grad, accumulate=grad0 is not None, **b, **size)
    else:
        hip.dispatch("distill_fwd", stats=stats, row_loss=row_loss, loss=loss, **b, **size)
        hip.dispatch("distill_bwd", stats=stats, grad=grad, accumulate=grad0 is not None, **b, **size)
    whole = hip.to_numpy(g)
    assert (whole[:guard] == 3.5).all() and (whole[-guard:] == 3.5).all()
    out = {"stats": hip.to_numpy(stats, (rows, 2)), "row_loss": hip.to_numpy(row_loss), "loss": float(hip.to_numpy(loss)[0]),
           "grad": whole[guard:-guard].reshape(rows, cols)}
    for buf in (*b.values(), stats, row_loss, loss, g):
        hip.mem_free(buf)
    return out


def check(got, x, teacher, indices, temp, weights=None, grad0=None):
    rows = x.shape[0]
    ref = distill(x, teacher, indices, temp, weights)
    w = np.full(rows, 1.0 / rows) if weights is None else weights.astype(np.float64)
    tol = distill_bounds(ref, np.where(w[:, None] != 0, x, 0), temp, w)
    assert np.array_equal(got["stats"][:, 0], ref["stats"][:, 0].astype(np.float32))
    assert (np.abs(got["stats"][:, 1] - ref["stats"][:, 1]) <= tol["ls"]).all()
    fine = np.isfinite(ref["row_loss"])
    assert np.array_equal(got["row_loss"][~fine], ref["row_loss"][~fine].astype(np.float32))
    assert (np.abs(got["row_loss"][fine] - ref["row_loss"][fine]) <= tol["row_loss"][fine]).all()
    if fine.all():
        assert abs(got["loss"] - ref["loss"]) <= (np.abs(w) * (tol["row_loss"] + (rows / 64 + 16) * EPS * np.abs(ref["row_loss"]))).sum()
    else:
        assert got["loss"] == np.inf
    want = ref["grad"] if grad0 is None else ref["grad"] + grad0.astype(np.float64)
    slack = tol["grad"] if grad0 is None else tol["grad"] + 2 * EPS * (np.abs(want) + np.abs(grad0))
    # products of probabilities below the smallest normal number lose bits: half a step of the smallest denormal, per factor
    assert (np.abs(got["grad"] - want) <= slack + 2.0**-126).all()
    return ref


SHAPES = [(1, 1, 1), (1, 2, 1), (3, 5, 5), (64, 10, 3), (5, 16, 8), (7, 33, 33), (100, 63, 7), (9, 64, 20), (4, 65, 65), (6, 255, 30),
          (5, 256, 100), (3, 257, 8), (2, 1000, 512), (4, 1023, 64), (3, 1025, 64), (2, 2047, 100), (3, 4095, 64), (2, 4097, 300),
          (2, 8191, 64), (1, 8193, 64), (3, 10007, 100), (2, 16384, 64), (2, 32000, 64), (3, 32769, 128), (2, 50257, 100), (1, 131075, 256)]


@pytest.mark.parametrize("rows,cols,k", SHAPES)
@pytest.mark.parametrize("fused", [False, True])
def test_every_row_length(hip, rows, cols, k, fused):
    x, teacher, indices, grad0 = case(rows + cols, rows, cols, k)
    for temp, add in ((1.0, None), (2.0, grad0)):
        check(run(hip, x, teacher, indices, temp, None, add, fused), x, teacher, indices, temp, None, add)


@pytest.mark.parametrize("rows,cols,k", [(3000, 10, 3), (70000, 3, 2), (1000, 100, 16), (2000, 1000, 64), (300, 5000, 64), (129, 32001, 64)])
@pytest.mark.parametrize("fused", [False, True])
def test_many_rows(hip, rows, cols, k, fused):
    x, teacher, indices, grad0 = case(rows, rows, cols, k)
    check(run(hip, x, teacher, indices, 2.0, None, grad0, fused), x, teacher, indices, 2.0, None, grad0)


@pytest.mark.parametrize("cols", [8192, 8196, 16385, 32764, 32768, 65532, 65536, 65537, 65541])
@pytest.mark.parametrize("fused", [False, True])
def test_row_lengths_around_the_kernels_own(hip, cols, fused):
    x, teacher, indices, grad0 = case(cols, 3, cols, 20)
    w = np.array([0.25, 0.0, 0.5], np.float32)
    for add in (None, grad0):
        check(run(hip, x, teacher, indices, 2.0, w, add, fused), x, teacher, indices, 2.0, w, add)


@pytest.mark.parametrize("cols", [257, 511, 512, 513, 1024, 2048, 2049, 4096, 4097, 16384])
@pytest.mark.parametrize("k", [64, 65, 257])
@pytest.mark.parametrize("fused", [False, True])
def test_numbers_of_entries(hip, cols, k, fused):
    x, teacher, indices, grad0 = case(cols + k, 3, cols, k)
    indices[1, 3:9] = indices[1, 2]  # one class seven times
    for add in (None, grad0):
        check(run(hip, x, teacher, indices, 1.5, None, add, fused), x, teacher, indices, 1.5, None, add)


@pytest.mark.parametrize("cols", [10, 200, 5000, 33000, 70000])
def test_extreme_temperatures(hip, cols):
    """At 1e-18 every row but those of equal logits has one class; at 1e18 all classes are equal and the loss is next to nothing."""
    x, teacher, indices, _ = case(cols, 3, cols, 4)
    x[:, :4], teacher[:], indices[:] = 0, 0, np.arange(4)
    x[:, 4:] = -1 - np.abs(x[:, 4:])
    for fused in (False, True):
        got = run(hip, x, teacher, indices, 1e-18, None, None, fused)
        assert (got["stats"][:, 0] == 0).all() and np.abs(got["stats"][:, 1] - np.log(4)).max() <= 4 * EPS * np.log(4)
        assert np.abs(got["row_loss"]).max() <= 1e-36 and np.abs(got["grad"][:, :4]).max() <= 1e-18
        assert (got["grad"][:, 4:] == 0).all()
        got = run(hip, x, teacher, indices, 1e18, None, None, fused)
        # gradient: temperature / rows (1 / cols - [kept] / 4).  p = exp(-log cols): the logarithm, its difference and the argument
        # of the exponential are off by 5 halves of a step of log cols together, the exponential and the factors by 8 of p;
        # q and its factors by 16 of q
        p, q = np.full((3, cols), 1 / cols), np.zeros((3, cols))
        q[:, :4] = 0.25
        slack = (p * (5 * np.log(cols) + 8) + 16 * q + 2 * np.abs(p - q)) * EPS
        assert (np.abs(got["grad"] / (1e18 / 3) - (p - q)) <= slack).all()


@pytest.mark.parametrize("temp", [0.05, 0.5, 1.0, 3.0, 20.0])
@pytest.mark.parametrize("cols", [12, 700, 9000])
def test_temperatures(hip, temp, cols):
    x, teacher, indices, _ = case(5, 6, cols, 9)
    for fused in (False, True):
        check(run(hip, x, teacher, indices, temp, fused=fused), x, teacher, indices, temp)


@pytest.mark.parametrize("cols", [10, 300, 5000, 40000])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("add", [False, True])
def test_padding_weights_and_empty_rows(hip, cols, fused, add):
    r = np.random.default_rng(cols)
    x, teacher, indices, grad0 = case(cols, 12, cols, 8)
    weights = r.random(12).astype(np.float32)
    weights[2] = weights[7] = 0
    x[2] = np.nan                       # a padding row holds anything
    teacher[7], indices[7] = np.nan, U64(2**64 - 1)
    x[3] = -np.inf                      # no class left
    x[4, : cols // 2] = -np.inf         # masked classes
    indices[4] = np.arange(8) + cols // 2 if cols >= 16 else cols - 1
    x[5] = np.finfo(np.float32).min     # masked by the lowest value throughout: uniform
    indices[6] = U64(2**64 - 1)         # nothing kept of the teacher
    teacher[8] = -np.inf
    teacher[9, 3:] = -np.inf            # kept, without weight
    indices[10, 1:] = indices[10, 0]    # one class several times
    indices[11, ::2] = U64(cols)        # padding among the kept
    grad0 = grad0 if add else None
    got = run(hip, x, teacher, indices, 2.0, weights, grad0, fused)
    ref = check(got, x, teacher, indices, 2.0, weights, grad0)
    for row in (2, 3, 6, 7, 8):
        assert got["row_loss"][row] == 0 and ref["row_loss"][row] == 0
        assert np.array_equal(got["grad"][row], grad0[row] if add else np.zeros(cols, np.float32))
    assert np.isfinite(got["loss"])


@pytest.mark.parametrize("cols", [10, 300, 5000])
@pytest.mark.parametrize("fused", [False, True])
def test_a_class_the_student_excludes_costs_everything(hip, cols, fused):
    x, teacher, indices, _ = case(1, 4, cols, 5)
    x[1, int(indices[1, 0])] = -np.inf
    got = run(hip, x, teacher, indices, 1.0, fused=fused)
    check(got, x, teacher, indices, 1.0)
    assert got["row_loss"][1] == np.inf and got["loss"] == np.inf and np.isfinite(got["grad"]).all()


@pytest.mark.parametrize("cols", [10, 300, 5000, 40000])
@pytest.mark.parametrize("fused", [False, True])
def test_a_nan_spoils_its_row_and_the_loss_only(hip, cols, fused):
    x, teacher, indices, _ = case(2, 5, cols, 5)
    x[1, cols - 1] = np.nan
    x[2] = -np.inf
    x[2, 0] = np.nan
    teacher[3, 4] = np.nan
    got = run(hip, x, teacher, indices, 1.0, fused=fused)
    bad = np.array([False, True, True, True, False])
    assert np.isnan(got["row_loss"][bad]).all() and np.isfinite(got["row_loss"][~bad]).all() and np.isnan(got["loss"])
    assert np.isnan(got["grad"][1:3]).all() and np.isfinite(got["grad"][~bad]).all()
    assert np.isnan(got["grad"][3][indices[3].astype(np.int64)]).all()


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_operands_off_the_16_byte_grid(hip, shift):
    for cols in (10, 64, 1000, 9001, 32768):
        x, teacher, indices, grad0 = case(cols, 5, cols, 8)
        pad = lambda a: hip.from_numpy(np.concatenate([np.zeros(shift, np.float32), a.ravel()])).sub(shift, a.size)  # noqa: E731
        for fused in (False, True):
            lb, tb, gb, ib = pad(x), pad(teacher), pad(grad0), hip.from_numpy(indices)
            stats, row_loss, loss = pad(np.zeros(10, np.float32)), pad(np.zeros(5, np.float32)), pad(np.zeros(1, np.float32))
            p = dict(logits=lb, teacher=tb, indices=ib, stats=stats, rows=5, cols=cols, k=8, temperature=2.0)
            if fused:
                hip.dispatch("distill_fwd_bwd", row_loss=row_loss, loss=loss, grad=gb, accumulate=True, **p)
            else:
                hip.dispatch("distill_fwd", row_loss=row_loss, loss=loss, **p)
                hip.dispatch("distill_bwd", grad=gb, accumulate=True, **p)
            got = {"stats": hip.to_numpy(stats, (5, 2)), "row_loss": hip.to_numpy(row_loss), "loss": float(hip.to_numpy(loss)[0]),
                   "grad": hip.to_numpy(gb, (5, cols))}
            check(got, x, teacher, indices, 2.0, None, grad0)


def test_the_same_bits_every_time_and_from_pinned_indices(hip):
    x, teacher, indices, grad0 = case(9, 40, 20000, 64)
    first = run(hip, x, teacher, indices, 2.0, None, grad0, True)
    again = run(hip, x, teacher, indices, 2.0, None, grad0, True)
    assert all(np.array_equal(first[n], again[n]) for n in ("stats", "row_loss", "grad")) and first["loss"] == again["loss"]
    pinned = hip.mem_alloc_host(np.uint64, indices.size)
    hip.host_view(pinned)[:] = indices.ravel()
    b = [hip.from_numpy(a) for a in (x, teacher, grad0)]
    out = [hip.mem_alloc(np.float32, n) for n in (80, 40, 1)]
    hip.dispatch("distill_fwd_bwd", logits=b[0], teacher=b[1], indices=pinned, stats=out[0], row_loss=out[1], loss=out[2], grad=b[2],
                 rows=40, cols=20000, k=64, temperature=2.0, accumulate=True)
    assert np.array_equal(hip.to_numpy(b[2], x.shape), first["grad"])
    for buf in (*b, *out, pinned):
        hip.mem_free(buf)


def test_the_formula_is_the_gradient_of_the_loss():
    """In 64 bits, central differences of step h: off by h^2 / 6 times the third derivative (at most 1 / T^2 here) and by the
    loss's rounding over h."""
    r = np.random.default_rng(4)
    x, t = r.standard_normal((3, 7)), r.standard_normal((3, 4))
    at, w = ((r.integers(0, 7, (3, 1)) + np.arange(4)) % 7).astype(U64), r.random(3)
    ref, h = distill(x, t, at, 2.0, w), 1e-4
    for row in range(3):
        for c in range(7):
            up, down = x.copy(), x.copy()
            up[row, c] += h
            down[row, c] -= h
            diff = (distill(up, t, at, 2.0, w)["loss"] - distill(down, t, at, 2.0, w)["loss"]) / (2 * h)
            assert abs(diff - ref["grad"][row, c]) <= h * h + 1e-14 / h
