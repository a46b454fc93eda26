"""Rows ordered by expert, laid out in that order and brought back with weights: the order exact, copies bit for bit, sums within
the roundings of their terms."""
import numpy as np
import pytest

from topk_reference import EPS, NONE, expert_sort, gather, spread

pytestmark = pytest.mark.gpu
U64 = np.uint64


def run_sort(hip, experts, n_experts, guard=32):
    n = len(experts)
    e = hip.from_numpy(experts)
    offsets, slots = (hip.from_numpy(np.full(m + 2 * guard, 77, U64)) for m in (n_experts + 1, n))
    hip.dispatch("expert_sort", experts=e, offsets=offsets.sub(guard, n_experts + 1), slots=slots.sub(guard, n), n_experts=n_experts)
    o, s = hip.to_numpy(offsets), hip.to_numpy(slots)
    for b in (e, offsets, slots):
        hip.mem_free(b)
    for a in (o, s):
        assert (a[:guard] == 77).all() and (a[len(a) - guard:] == 77).all()
    return o[guard:-guard], s[guard:-guard]


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 511, 512, 513, 1000, 4096, 8191, 8192, 8193, 9000, 65536, 100003, 300000])
@pytest.mark.parametrize("n_experts", [1, 2, 8, 63, 64, 65, 256, 1000, 1024])
def test_entries_are_ordered_by_expert_first_come_first(hip, n, n_experts):
    r = np.random.default_rng(n + n_experts)
    kinds = [r.integers(0, n_experts, n), np.minimum(r.geometric(0.3, n) - 1, n_experts), np.full(n, n_experts - 1)]
    for experts in kinds:
        experts = experts.astype(U64)
        if n > 2:
            experts[r.random(n) < 0.1] = U64(n_experts)     # dropped, in three ways
            experts[0], experts[n // 2] = NONE, U64(1 << 32)
        o, s = run_sort(hip, experts, n_experts)
        want_o, want_s = expert_sort(experts, n_experts)
        assert np.array_equal(o, want_o) and np.array_equal(s, want_s)


def test_no_entry_is_held(hip):
    for n in (5, 20000):
        o, s = run_sort(hip, np.full(n, 9, U64), 4)
        assert (o == 0).all() and (s == NONE).all()


def layout(seed, tokens, k, n_experts):
    r = np.random.default_rng(seed)
    experts = np.argsort(r.random((tokens, n_experts)) + 2 * r.random(n_experts), axis=1)[:, :k].astype(U64)
    experts[r.random((tokens, k)) < 0.1] = U64(n_experts)
    if tokens > 2:
        experts[1] = U64(n_experts)  # a token that goes nowhere
    _, slots = expert_sort(experts.ravel(), n_experts)
    return r, slots


def guarded(hip, a, guard=16):
    return hip.from_numpy(np.concatenate([np.full(guard, 3.5, np.float32), a.ravel(), np.full(guard, 3.5, np.float32)])), guard


def read(hip, buf, guard, shape):
    a = hip.to_numpy(buf)
    assert (a[:guard] == 3.5).all() and (a[-guard:] == 3.5).all()
    return a[guard:-guard].reshape(shape)


TOKENS = [(1, 1, 1, 1), (1, 2, 4, 7), (3, 1, 2, 16), (5, 3, 8, 33), (64, 2, 8, 64), (100, 8, 16, 100), (33, 6, 64, 130), (257, 4, 8, 255),
          (17, 7, 7, 1024), (50, 2, 4, 1030), (9, 64, 64, 40), (2, 3, 8, 5000), (700, 2, 300, 36), (1000, 8, 32, 260)]


@pytest.mark.parametrize("tokens,k,n_experts,width", TOKENS)
@pytest.mark.parametrize("shift", [0, 1])
def test_rows_go_to_their_places_and_back(hip, tokens, k, n_experts, width, shift):
    """shift: every array begins one value off the 16-byte grid."""
    r, slots = layout(tokens + k, tokens, k, n_experts)
    n, guard = tokens * k, 16 + shift
    x, y = r.standard_normal((tokens, width)).astype(np.float32), r.standard_normal((n, width)).astype(np.float32)
    w, base = r.standard_normal((tokens, k)).astype(np.float32), r.standard_normal((n, width)).astype(np.float32)
    y[np.setdiff1d(np.arange(n), slots[slots != NONE].astype(np.int64))] = np.nan  # rows behind the last place are not read
    bufs = {"slots": hip.from_numpy(slots), "w": hip.from_numpy(w)}
    put = lambda name, a: bufs.setdefault(name, guarded(hip, a, guard)[0]).sub(guard, a.size)  # noqa: E731
    size = dict(n_tokens=tokens, k=k, width=width)
    xv, yv, ov = put("x", x), put("y", y), put("out", np.zeros((tokens, width), np.float32))
    rows_v, yg_v, wg_v = put("rows", base), put("y_g", base), put("w_g", np.zeros((tokens, k), np.float32))
    xg_v = put("x_g", x)
    hip.dispatch("expert_dispatch", x=xv, slots=bufs["slots"], y=rows_v, **size)
    assert np.array_equal(read(hip, bufs["rows"], guard, (n, width)), spread(x, slots, k, base).astype(np.float32))

    hip.dispatch("expert_combine", y=yv, slots=bufs["slots"], weights=bufs["w"], out=ov, **size)
    want, scale = gather(y, slots, tokens, k, w)
    got = read(hip, bufs["out"], guard, (tokens, width))
    assert (np.abs(got - want) <= (k + 1) * EPS * scale).all()     # a product and k - 1 sums
    assert (got[scale == 0] == 0).all()

    for accumulate in (True, False):
        hip.dispatch("expert_dispatch_bwd", y_g=yv, slots=bufs["slots"], x_g=xg_v, accumulate=accumulate, **size)
        want, scale = gather(y, slots, tokens, k)
        if accumulate:
            want, scale = want + x, scale + np.abs(x)
        assert (np.abs(read(hip, bufs["x_g"], guard, (tokens, width)) - want) <= (k + 1) * EPS * scale).all()

    hip.dispatch("expert_combine_bwd", out_g=xv, y=yv, slots=bufs["slots"], weights=bufs["w"], y_g=yg_v, weights_g=wg_v, **size)
    want = spread(x, slots, k, base, w)
    got = read(hip, bufs["y_g"], guard, (n, width))
    assert (np.abs(got - want) <= EPS * np.abs(want)).all()        # one product
    places = slots.reshape(tokens, k)
    got = read(hip, bufs["w_g"], guard, (tokens, k))
    for t in range(tokens):
        for j in range(k):
            if places[t, j] == NONE:
                assert got[t, j] == 0
            else:
                terms = x[t].astype(np.float64) * y[int(places[t, j])].astype(np.float64)
                # a product each, and no term passes through more than width / 64 + 12 sums
                assert abs(got[t, j] - terms.sum()) <= (width / 64 + 14) * EPS * np.abs(terms).sum()
    for b in bufs.values():
        hip.mem_free(b)


def test_the_backward_of_the_combination_in_halves(hip):
    r, slots = layout(5, 40, 3, 8)
    x, y, w = (r.standard_normal(s).astype(np.float32) for s in ((40, 70), (120, 70), (40, 3)))
    size = dict(n_tokens=40, k=3, width=70)
    b = {n: hip.from_numpy(a) for n, a in (("x", x), ("y", y), ("w", w), ("slots", slots))}
    outs = []
    for want_y, want_w in ((True, True), (True, False), (False, True), (False, False)):
        y_g, w_g = hip.from_numpy(np.zeros_like(y)), hip.from_numpy(np.full_like(w, 5.0))
        hip.dispatch("expert_combine_bwd", out_g=b["x"], y=b["y"] if want_w else None, slots=b["slots"], weights=b["w"],
                     y_g=y_g if want_y else None, weights_g=w_g if want_w else None, **size)
        outs.append((hip.to_numpy(y_g), hip.to_numpy(w_g)))
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][1], outs[2][1])
    assert (outs[3][0] == 0).all() and (outs[3][1] == 5).all() and (outs[2][0] == 0).all() and (outs[1][1] == 5).all()


def test_slots_outside_the_rows_count_as_dropped(hip):
    slots = np.array([0, 6, 2, 1 << 40, NONE, 1], U64)
    x = np.arange(12, dtype=np.float32).reshape(3, 4)
    xb, sb, yb, wb = hip.from_numpy(x), hip.from_numpy(slots), hip.from_numpy(np.full((6, 4), -1, np.float32)), hip.from_numpy(np.ones(6, np.float32))
    size = dict(n_tokens=3, k=2, width=4)
    hip.dispatch("expert_dispatch", x=xb, slots=sb, y=yb, **size)
    want = np.full((6, 4), -1, np.float32)
    want[0], want[2], want[1] = x[0], x[1], x[2]
    assert np.array_equal(hip.to_numpy(yb, (6, 4)), want)
    ob = hip.from_numpy(np.full((3, 4), 9, np.float32))
    hip.dispatch("expert_combine", y=yb, slots=sb, weights=wb, out=ob, **size)
    assert np.array_equal(hip.to_numpy(ob, (3, 4)), x)


@pytest.mark.parametrize("tokens,k,n_experts,width", [(20000, 4, 64, 64), (3000, 8, 256, 1000), (70000, 1, 16, 12)])
def test_many_tokens_through_the_library_alone(hip, tokens, k, n_experts, width):
    """Sorted, laid out and summed with weights of powers of two: every token is its own row times its held weights."""
    r = np.random.default_rng(tokens)
    experts = r.integers(0, n_experts + 1, (tokens, k)).astype(U64)
    x, w = r.integers(-8, 9, (tokens, width)).astype(np.float32), (2.0 ** r.integers(-3, 1, (tokens, k))).astype(np.float32)
    eb, xb, wb = hip.from_numpy(experts.ravel()), hip.from_numpy(x), hip.from_numpy(w)
    off, slots = hip.mem_alloc(U64, n_experts + 1), hip.mem_alloc(U64, tokens * k)
    rows, out = hip.mem_alloc(np.float32, tokens * k * width), hip.mem_alloc(np.float32, tokens * width)
    size = dict(n_tokens=tokens, k=k, width=width)
    hip.dispatch("expert_sort", experts=eb, offsets=off, slots=slots, n_experts=n_experts)
    hip.dispatch("expert_dispatch", x=xb, slots=slots, y=rows, **size)
    hip.dispatch("expert_combine", y=rows, slots=slots, weights=wb, out=out, **size)
    held = (w * (experts < n_experts)).sum(axis=1, keepdims=True)
    assert np.array_equal(hip.to_numpy(out, (tokens, width)), x * held)
    want_o, want_s = expert_sort(experts.ravel(), n_experts)
    assert np.array_equal(hip.to_numpy(off), want_o) and np.array_equal(hip.to_numpy(slots), want_s)
    for b in (eb, xb, wb, off, slots, rows, out):
        hip.mem_free(b)
