"""Selection of the k largest of a row and its gradient: values, columns, order among equals, special values, every row
length and k at which the kernels change, all exact (nothing is rounded but the sums of repeated indices)."""
import numpy as np
import pytest

from topk_reference import EPS, topk, topk_bwd

pytestmark = pytest.mark.gpu
U64 = np.uint64


def run_fwd(hip, x, k, guard=64):
    """values and indices of x's rows; the words around the outputs must stay as they were."""
    rows, cols = x.shape
    xb = hip.from_numpy(x)
    v = hip.from_numpy(np.full(rows * k + 2 * guard, 7.5, np.float32))
    i = hip.from_numpy(np.full(rows * k + 2 * guard, 77, U64))
    hip.dispatch("topk_fwd", x=xb, values=v.sub(guard, rows * k), indices=i.sub(guard, rows * k), rows=rows, cols=cols, k=k)
    values, indices = hip.to_numpy(v), hip.to_numpy(i)
    for b in (xb, v, i):
        hip.mem_free(b)
    for a, mark in ((values, 7.5), (indices, 77)):
        assert (a[:guard] == mark).all() and (a[len(a) - guard:] == mark).all()
    return values[guard:-guard].reshape(rows, k), indices[guard:-guard].reshape(rows, k)


def check(hip, x, k):
    values, indices = run_fwd(hip, x, k)
    want_v, want_i = topk(x, k)
    assert np.array_equal(indices, want_i)
    assert np.array_equal(values.view(np.uint32), want_v.view(np.uint32))


COLS = [1, 2, 3, 5, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 250, 256, 257, 511, 512, 513, 1000, 1023, 1024, 1025, 2047, 2048, 2049,
        4095, 4097, 8191, 8192, 8193, 10000, 16385, 32001, 50257]


@pytest.mark.parametrize("cols", COLS)
def test_every_row_length(hip, cols):
    r = np.random.default_rng(cols)
    for rows in (1, 7):
        x = r.standard_normal((rows, cols)).astype(np.float32)
        for k in sorted({1, 2, min(cols, 8), min(cols, 33), min(cols, 100), min(cols, 512)}):
            if k <= cols:
                check(hip, x, k)


@pytest.mark.parametrize("k", [1, 2, 3, 4, 7, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512])
def test_every_k(hip, k):
    r = np.random.default_rng(k)
    for cols in (k, 600, 5000):
        if k <= cols:
            check(hip, r.standard_normal((5, cols)).astype(np.float32), k)


@pytest.mark.parametrize("cols,k", [(64, 8), (300, 40), (2048, 64), (9000, 100), (33000, 512)])
def test_equal_values_come_in_the_order_of_their_columns(hip, cols, k):
    r = np.random.default_rng(1)
    check(hip, np.zeros((3, cols), np.float32), k)
    check(hip, r.integers(0, 3, (4, cols)).astype(np.float32), k)
    check(hip, r.integers(0, max(2, cols // 4), (4, cols)).astype(np.float32), k)
    zeros = np.where(r.random((4, cols)) < 0.5, np.float32(0), np.float32(-0.0)).astype(np.float32)
    check(hip, zeros, k)
    one = np.full((2, cols), -np.inf, np.float32)
    one[0, cols - 1] = one[1, cols // 2] = -1
    check(hip, one, k)


@pytest.mark.parametrize("cols,k", [(100, 10), (1024, 64), (20000, 64), (20000, 300), (40000, 512)])
def test_sorted_rows(hip, cols, k):
    up = np.arange(cols, dtype=np.float32)
    stride = np.roll(up.reshape(-1, 4 if cols % 4 == 0 else 1), 1, axis=0).T.ravel()
    far = np.where(np.arange(cols) % 256 == 3, up + 1e6, up).astype(np.float32)  # the largest in one place of every 256
    check(hip, np.stack([up, up[::-1], -up, stride, far]), k)


@pytest.mark.parametrize("cols,k", [(20, 5), (64, 64), (700, 20), (5000, 64), (30000, 64)])
def test_special_values(hip, cols, k):
    r = np.random.default_rng(cols)
    x = r.standard_normal((8, cols)).astype(np.float32)
    x[0, r.random(cols) < 0.1] = np.nan
    x[1] = np.nan
    x[2, r.random(cols) < 0.2] = np.inf
    x[3, r.random(cols) < 0.9] = -np.inf
    x[4] = -np.inf
    x[5, r.random(cols) < 0.5] = np.finfo(np.float32).min
    x[6] = (r.integers(-5, 6, cols) * 1e-45).astype(np.float32)   # denormals
    x[7, -1] = -np.float32(np.nan)
    x[7, 0] = np.inf
    values, indices = run_fwd(hip, x, k)
    want_v, want_i = topk(x, k)
    assert np.array_equal(indices, want_i)
    assert np.array_equal(values, want_v, equal_nan=True)


@pytest.mark.parametrize("rows,cols,k", [(70000, 8, 2), (5000, 64, 8), (3000, 256, 8), (1000, 1000, 64), (300, 32000, 64), (2, 300000, 100)])
def test_many_rows(hip, rows, cols, k):
    x = np.random.default_rng(rows).standard_normal((rows, cols)).astype(np.float32)
    values, indices = run_fwd(hip, x, k)
    want = np.argsort(-x, axis=1, kind="stable")[:, :k] if cols <= 1000 else np.stack([np.argsort(-v, kind="stable")[:k] for v in x])
    assert np.array_equal(indices, want.astype(U64))
    assert np.array_equal(values, np.take_along_axis(x, want, axis=1))


@pytest.mark.parametrize("cols", [2049, 4100, 9003])
@pytest.mark.parametrize("k", [1, 40, 128])
def test_many_long_rows_of_every_kind(hip, cols, k):
    """Rows enough for the variant that gives a wave a row: eight kinds of row, each many times, in a mixed order."""
    r = np.random.default_rng(cols + k)
    kinds = [r.standard_normal(cols), np.arange(cols), -np.arange(cols), np.zeros(cols), r.integers(0, 5, cols),
             np.where(r.random(cols) < 0.5, np.inf, -np.inf), np.where(r.random(cols) < 0.01, np.nan, r.standard_normal(cols)),
             np.where(np.arange(cols) % 64 == 5, 1e3 + np.arange(cols), r.standard_normal(cols))]
    kinds = np.stack(kinds).astype(np.float32)
    which = r.integers(0, len(kinds), 4200)
    values, indices = run_fwd(hip, kinds[which], k)
    want_v, want_i = topk(kinds, k)
    assert np.array_equal(indices, want_i[which])
    assert np.array_equal(values, want_v[which], equal_nan=True)


@pytest.mark.parametrize("cols", [1, 4, 5, 16, 17, 60, 64, 100, 128, 131, 256])
def test_short_rows_of_every_kind(hip, cols):
    r = np.random.default_rng(cols)
    x = r.standard_normal((300, cols)).astype(np.float32)
    x[::3] = r.integers(-1, 2, (100, cols)) * np.float32(-0.0 if cols % 2 else 1.0)
    x[1::7, r.random(cols) < 0.3] = np.nan
    x[2::5, r.random(cols) < 0.5] = -np.inf
    for k in sorted({1, min(cols, 2), min(cols, 9), min(cols, 16), min(cols, 17), cols}):
        values, indices = run_fwd(hip, x, k)
        want_v, want_i = topk(x, k)
        assert np.array_equal(indices, want_i)
        assert np.array_equal(values, want_v, equal_nan=True)


@pytest.mark.parametrize("shift", [1, 2, 3])
def test_rows_off_the_16_byte_grid(hip, shift):
    r = np.random.default_rng(shift)
    for cols, k in ((64, 4), (1000, 20), (9001, 64)):
        x = r.standard_normal((6, cols)).astype(np.float32)
        xb = hip.from_numpy(np.concatenate([np.full(shift, 1e30, np.float32), x.ravel(), np.full(8, 1e30, np.float32)]))
        v, i = hip.from_numpy(np.zeros(6 * k + 1, np.float32)), hip.from_numpy(np.zeros(6 * k, U64))
        hip.dispatch("topk_fwd", x=xb.sub(shift, x.size), values=v.sub(1, 6 * k), indices=i, rows=6, cols=cols, k=k)
        want_v, want_i = topk(x, k)
        assert np.array_equal(hip.to_numpy(i).reshape(6, k), want_i)
        assert np.array_equal(hip.to_numpy(v)[1:].reshape(6, k), want_v)
        for b in (xb, v, i):
            hip.mem_free(b)


@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (3, 5, 2), (64, 64, 2), (100, 10, 10), (1000, 256, 8), (9, 1000, 512), (5, 32001, 64),
                                         (33, 129, 40), (70001, 4, 1), (2, 100003, 100)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_the_gradient_goes_to_the_chosen_places(hip, rows, cols, k, accumulate):
    r = np.random.default_rng(rows + cols)
    start = r.integers(0, cols, (rows, 1))
    indices = ((start + np.arange(k) * 3) % cols if np.gcd(3, cols) == 1 else (start + np.arange(k)) % cols).astype(U64)
    y_g, x_g = r.standard_normal((rows, k)).astype(np.float32), r.standard_normal((rows, cols)).astype(np.float32)
    got = run_bwd(hip, indices, y_g, x_g, accumulate)
    want = x_g.copy() if accumulate else np.zeros_like(x_g)
    at = indices.astype(np.int64)
    if min(k, cols) == k:  # no index twice: one rounding
        np.put_along_axis(want, at, np.take_along_axis(want, at, axis=1) + y_g, axis=1)
        assert np.array_equal(got, want)


def run_bwd(hip, indices, y_g, x_g, accumulate, guard=64):
    rows, cols = x_g.shape
    ib, yb = hip.from_numpy(indices), hip.from_numpy(y_g)
    xb = hip.from_numpy(np.concatenate([np.full(guard, 3.5, np.float32), x_g.ravel(), np.full(guard, 3.5, np.float32)]))
    hip.dispatch("topk_bwd", indices=ib, y_g=yb, x_g=xb.sub(guard, x_g.size), rows=rows, cols=cols, k=indices.shape[1],
                 accumulate=accumulate)
    out = hip.to_numpy(xb)
    for b in (ib, yb, xb):
        hip.mem_free(b)
    assert (out[:guard] == 3.5).all() and (out[-guard:] == 3.5).all()
    return out[guard:-guard].reshape(rows, cols)


@pytest.mark.parametrize("cols,k", [(3, 20), (50, 64), (300, 400), (2000, 512)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_repeated_and_padding_indices_in_the_gradient(hip, cols, k, accumulate):
    """An index may stand in a row several times (its gradients are added in the order of j: at most k roundings) or lie
    outside the row (it takes part in nothing)."""
    r = np.random.default_rng(k)
    indices = r.integers(0, cols, (20, k)).astype(U64)
    indices[r.random((20, k)) < 0.2] = U64(2**64 - 1)
    indices[r.random((20, k)) < 0.1] = U64(cols)
    indices[3] = U64(2**33)
    y_g, x_g = r.standard_normal((20, k)).astype(np.float32), r.standard_normal((20, cols)).astype(np.float32)
    got = run_bwd(hip, indices, y_g, x_g, accumulate)
    base = x_g if accumulate else np.zeros_like(x_g)
    want, size = topk_bwd(indices, y_g, base), topk_bwd(indices, np.abs(y_g), np.abs(base))
    assert (np.abs(got - want) <= k * EPS * size).all()
    assert np.array_equal(run_bwd(hip, indices, y_g, x_g, accumulate), got)


def test_the_gradient_of_a_selection_is_what_differences_say(hip):
    """sum(g * topk(x)) moves by g_j when the j-th largest moves: in steps that change no order, exact in powers of two."""
    r = np.random.default_rng(3)
    x = r.permutation(40).astype(np.float32).reshape(1, 40)
    g = r.integers(-8, 9, (1, 6)).astype(np.float32)
    _, indices = run_fwd(hip, x, 6)
    grad = run_bwd(hip, indices, g, np.zeros_like(x), False)
    for c in range(40):
        up, down = x.copy(), x.copy()
        up[0, c] += 0.25
        down[0, c] -= 0.25
        diff = ((run_fwd(hip, up, 6)[0] - run_fwd(hip, down, 6)[0]) * g).sum() / 0.5
        assert diff == grad[0, c]
