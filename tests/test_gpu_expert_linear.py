"""The experts' Linear layers against products in 64 bits: ranges of every length, none among them, odd layer sizes, operands off
the 16-byte grid, rows behind the last expert untouched.  A dot product of n terms in fp32 is off by at most n + 2 halves of
a step of the sum of the terms' magnitudes, in any order of the sums."""
import numpy as np
import pytest

from topk_reference import EPS

pytestmark = pytest.mark.gpu
U64 = np.uint64
GUARD = 32


def offsets_of(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(U64)


def put(hip, a, shift=0):
    buf = hip.from_numpy(np.concatenate([np.full(GUARD + shift, 3.5, np.float32), a.ravel(), np.full(GUARD, 3.5, np.float32)]))
    return buf, buf.sub(GUARD + shift, a.size)


def get(hip, buf, shift, shape):
    a = hip.to_numpy(buf)
    assert (a[: GUARD + shift] == 3.5).all() and (a[-GUARD:] == 3.5).all()
    return a[GUARD + shift: -GUARD].reshape(shape)


def case(seed, counts, behind, fan_in, fan_out):
    r = np.random.default_rng(seed)
    n, e = int(np.sum(counts)) + behind, len(counts)
    return {"x": r.standard_normal((n, fan_in)).astype(np.float32), "w": r.standard_normal((e, fan_out, fan_in)).astype(np.float32),
            "b": r.standard_normal((e, fan_out)).astype(np.float32), "gy": r.standard_normal((n, fan_out)).astype(np.float32),
            "act": np.maximum(r.standard_normal((n, fan_in)), 0).astype(np.float32), "offsets": offsets_of(counts),
            "n": n, "e": e, "i": fan_in, "o": fan_out}


def check_fwd(hip, c, bias, relu, shift=0):
    n, e, i, o = c["n"], c["e"], c["i"], c["o"]
    x = c["x"].copy()
    x[int(c["offsets"][-1]):] = np.nan  # rows behind the last expert are not read
    xb, wb, bb, yb = put(hip, x, shift), put(hip, c["w"], shift), put(hip, c["b"], shift), put(hip, np.full((n, o), 9, np.float32), shift)
    off = hip.from_numpy(c["offsets"])
    hip.dispatch("expert_linear_fwd", x=xb[1], w=wb[1], bias=bb[1] if bias else None, y=yb[1], offsets=off, n_rows=n, n_experts=e,
                 fan_in=i, fan_out=o, relu=relu)
    y = get(hip, yb[0], shift, (n, o))
    for k in range(e):
        s = slice(int(c["offsets"][k]), int(c["offsets"][k + 1]))
        a, m = c["x"][s].astype(np.float64), c["w"][k].astype(np.float64).T
        want, size = a @ m, np.abs(a) @ np.abs(m)
        if bias:
            want, size = want + c["b"][k], size + np.abs(c["b"][k])
        want = np.maximum(want, 0) if relu else want
        assert (np.abs(y[s] - want) <= (i + 3) * EPS * size).all(), k
    assert (y[int(c["offsets"][-1]):] == 9).all()
    for b in (xb[0], wb[0], bb[0], yb[0], off):
        hip.mem_free(b)


def check_bwd(hip, c, bias, mask, accumulate, shift=0, want_gx=True):
    n, e, i, o = c["n"], c["e"], c["i"], c["o"]
    r = np.random.default_rng(1)
    gw0, gb0 = r.standard_normal((e, o, i)).astype(np.float32), r.standard_normal((e, o)).astype(np.float32)
    x, gy = c["x"].copy(), c["gy"].copy()
    last = int(c["offsets"][-1])
    x[last:] = gy[last:] = np.nan
    b = {"gy": put(hip, gy, shift), "x": put(hip, x, shift), "w": put(hip, c["w"], shift), "act_in": put(hip, c["act"], shift),
         "gw": put(hip, gw0, shift), "gb": put(hip, gb0, shift), "gx": put(hip, np.full((n, i), 9, np.float32), shift)}
    off = hip.from_numpy(c["offsets"])
    hip.dispatch("expert_linear_bwd", gy=b["gy"][1], x=b["x"][1], w=b["w"][1], act_in=b["act_in"][1] if mask else None, gw=b["gw"][1],
                 gb=b["gb"][1] if bias else None, gx=b["gx"][1] if want_gx else None, offsets=off, n_rows=n, n_experts=e, fan_in=i,
                 fan_out=o, accumulate=accumulate)
    gw, gb, gx = get(hip, b["gw"][0], shift, (e, o, i)), get(hip, b["gb"][0], shift, (e, o)), get(hip, b["gx"][0], shift, (n, i))
    for k in range(e):
        s = slice(int(c["offsets"][k]), int(c["offsets"][k + 1]))
        g, a, m = c["gy"][s].astype(np.float64), c["x"][s].astype(np.float64), c["w"][k].astype(np.float64)
        rows = g.shape[0]
        for got, first, want, size in ((gw[k], gw0[k], g.T @ a, np.abs(g).T @ np.abs(a)), (gb[k], gb0[k], g.sum(0), np.abs(g).sum(0))):
            if got is gb[k] or got.ndim == 1:
                if not bias:
                    assert np.array_equal(got, first)
                    continue
            if accumulate:
                want, size = want + first, size + np.abs(first)
            assert (np.abs(got - want) <= (rows + 3) * EPS * size).all(), k
        if want_gx:
            want, size = g @ m, np.abs(g) @ np.abs(m)
            if mask:
                want, size = want * (c["act"][s] > 0), size * (c["act"][s] > 0)
            assert (np.abs(gx[s] - want) <= (o + 3) * EPS * size).all(), k
    assert (gx[last:] == 9).all() and (want_gx or (gx == 9).all())
    for buf, _ in b.values():
        hip.mem_free(buf)
    hip.mem_free(off)


CASES = [([1], 0, 1, 1), ([3], 2, 5, 7), ([0, 1], 0, 16, 16), ([5, 0, 3], 1, 33, 17), ([64, 64], 0, 64, 64), ([1, 2, 3, 4, 0, 6, 7], 3, 100, 30),
         ([130, 5, 0, 64, 63, 65], 7, 96, 130), ([17] * 8, 0, 250, 255), ([300, 2], 10, 128, 64), ([0, 0, 0], 5, 40, 24), ([200, 100, 411], 0, 1000, 66),
         ([1, 1, 1, 1], 0, 1024, 512), ([8, 9, 40, 31], 4, 515, 129), ([700], 0, 36, 260), ([0, 2000, 1, 0], 0, 65, 68), ([16, 15, 1, 32, 33, 0, 48], 2, 260, 196)]


@pytest.mark.parametrize("counts,behind,fan_in,fan_out", CASES)
@pytest.mark.parametrize("shift", [0, 1])
def test_forward(hip, counts, behind, fan_in, fan_out, shift):
    c = case(len(counts) + fan_in, counts, behind, fan_in, fan_out)
    for bias, relu in ((False, False), (True, True)):
        check_fwd(hip, c, bias, relu, shift)


@pytest.mark.parametrize("counts,behind,fan_in,fan_out", CASES)
@pytest.mark.parametrize("shift", [0, 1])
def test_backward(hip, counts, behind, fan_in, fan_out, shift):
    c = case(len(counts) + fan_in, counts, behind, fan_in, fan_out)
    for bias, mask, accumulate in ((True, True, True), (False, False, False), (True, False, False)):
        check_bwd(hip, c, bias, mask, accumulate, shift)
    check_bwd(hip, c, True, False, True, shift, want_gx=False)


@pytest.mark.parametrize("n_experts", [63, 64, 65, 130, 1024])
def test_many_experts(hip, n_experts):
    r = np.random.default_rng(n_experts)
    counts = np.where(r.random(n_experts) < 0.4, 0, r.integers(1, 9, n_experts))
    counts[n_experts // 2] = 200
    c = case(n_experts, counts, 9, 36, 40)
    check_fwd(hip, c, True, False)
    check_bwd(hip, c, True, True, True)


@pytest.mark.parametrize("n,e,fan_in,fan_out", [(5000, 16, 256, 384), (3000, 3, 512, 300), (9000, 40, 130, 128)])
def test_ordinary_layers(hip, n, e, fan_in, fan_out):
    r = np.random.default_rng(n)
    share = r.random(e) ** 3
    counts = np.floor(share / share.sum() * (n - 20)).astype(int)
    c = case(n, counts, n - int(counts.sum()), fan_in, fan_out)
    check_fwd(hip, c, True, True)
    check_bwd(hip, c, True, True, False)


@pytest.mark.parametrize("n_experts,per,fan_in,fan_out", [(65, 12, 50, 70), (1024, 10, 17, 33), (24, 12, 1020, 1024), (67, 9, 637, 640)])
def test_many_experts_of_many_rows(hip, n_experts, per, fan_in, fan_out):
    """The experts' order found by a launch of its own (more than 64), the large tiles of the weight gradients."""
    r = np.random.default_rng(n_experts)
    counts = r.integers(0, 2 * per, n_experts)
    counts[::5] = 0
    counts[1] += 3 * per
    counts[0] = max(0, n_experts * per - int(counts.sum()))
    c = case(n_experts, counts, 1, fan_in, fan_out)
    assert c["n"] // n_experts > 8
    check_fwd(hip, c, True, True)
    check_bwd(hip, c, True, True, True)
    check_bwd(hip, c, False, False, False, shift=1)


@pytest.mark.parametrize("counts,behind,fan_in,fan_out", [([515], 0, 20, 30), ([4000], 3, 64, 130), ([3000, 0, 1], 5, 96, 63), ([0, 2500, 900], 0, 17, 70),
                                                          ([34000] + [1, 0, 5] * 21 + [40], 2, 20, 12), ([129] * 3 + [2000], 0, 260, 65)])
def test_small_layers_with_many_rows(hip, counts, behind, fan_in, fan_out):
    """The rows of an expert in parts for its weight gradient, added up afterwards; parts without a row."""
    c = case(len(counts) + fan_in, counts, behind, fan_in, fan_out)
    check_fwd(hip, c, True, True)
    for bias, mask, accumulate in ((True, True, True), (False, False, False)):
        check_bwd(hip, c, bias, mask, accumulate, shift=1 if accumulate else 0)


@pytest.mark.parametrize("rows", [1, 17, 40, 100, 250, 1030])
@pytest.mark.parametrize("fan_in,fan_out", [(100, 260), (1030, 64), (64, 1000)])
def test_one_expert(hip, rows, fan_in, fan_out):
    c = case(rows, [rows], 1, fan_in, fan_out)
    check_fwd(hip, c, True, True)
    check_bwd(hip, c, True, True, True)


@pytest.mark.parametrize("n,e,fan_in,fan_out", [(4500, 70, 68, 1920), (10500, 5, 302, 1660), (2700, 3, 200, 6143)])
def test_wide_tiles(hip, n, e, fan_in, fan_out):
    """Enough tiles of 64 x 128 for all compute units, forward or in the input gradient, the last column of tiles whole or not."""
    r = np.random.default_rng(n)
    share = r.random(e) ** 2
    counts = np.floor(share / share.sum() * (n - 7)).astype(int)
    c = case(n, counts, n - int(counts.sum()), fan_in, fan_out)
    check_fwd(hip, c, True, True)
    check_fwd(hip, c, True, False, shift=1)
    c = case(n + 1, counts, n - int(counts.sum()), fan_out, fan_in)
    check_bwd(hip, c, True, True, False)
    check_bwd(hip, c, False, False, True, shift=3)


@pytest.mark.parametrize("per", [2, 3, 6, 7, 16, 17, 20, 21, 32, 33, 48, 49])
@pytest.mark.parametrize("n_experts,fan_in,fan_out", [(8, 64, 96), (16, 520, 260), (40, 96, 516)])
def test_rows_per_expert(hip, n_experts, fan_in, fan_out, per):
    """The average number of rows decides between the kernels for few rows and the tiled ones; some experts have other numbers."""
    r = np.random.default_rng(per)
    counts = np.full(n_experts, per)
    counts[1], counts[3] = 0, 2 * per
    counts[5:8] = r.multinomial(3 * per, [0.7, 0.2, 0.1])
    c = case(per, counts, 0, fan_in, fan_out)
    check_fwd(hip, c, True, True)
    check_bwd(hip, c, True, True, True, shift=per % 2)


@pytest.mark.parametrize("counts,fan_in,fan_out", [([3, 5, 2, 4], 40, 36), ([30, 21, 50, 18], 70, 66), ([300, 120, 500, 200], 132, 200)])
def test_one_expert_of_nan_leaves_the_others_alone(hip, counts, fan_in, fan_out):
    c = case(5, counts, 0, fan_in, fan_out)
    offsets = c["offsets"].astype(int)
    bad = slice(offsets[2], offsets[3])
    out = {}
    for kind in ("clean", "nan"):
        if kind == "nan":
            c["x"][bad], c["gy"][bad], c["w"][2], c["b"][2] = np.nan, np.inf, -np.inf, np.nan
        b = {n: hip.from_numpy(c[n]) for n in ("x", "w", "b", "gy", "act", "offsets")}
        y, gw, gb, gx = (hip.from_numpy(np.zeros(s, np.float32)) for s in (c["gy"].shape, c["w"].shape, c["b"].shape, c["x"].shape))
        layer = dict(offsets=b["offsets"], n_rows=c["n"], n_experts=4, fan_in=fan_in, fan_out=fan_out)
        hip.dispatch("expert_linear_fwd", x=b["x"], w=b["w"], bias=b["b"], y=y, relu=False, **layer)
        hip.dispatch("expert_linear_bwd", gy=b["gy"], x=b["x"], w=b["w"], act_in=b["act"], gw=gw, gb=gb, gx=gx, accumulate=False, **layer)
        out[kind] = [hip.to_numpy(y, c["gy"].shape), hip.to_numpy(gw, c["w"].shape), hip.to_numpy(gb, c["b"].shape), hip.to_numpy(gx, c["x"].shape)]
    others = np.ones(c["n"], bool)
    others[bad] = False
    for i, (clean, nan) in enumerate(zip(out["clean"], out["nan"])):
        keep = others if i in (0, 3) else np.array([True, True, False, True])
        assert np.array_equal(clean[keep], nan[keep]), i
        assert not np.isfinite(nan[~keep]).all(), i


def test_offsets_that_make_no_sense_stay_inside_the_rows(hip):
    """Ranges beyond n_rows end there, ranges that end before they begin are empty."""
    c = case(3, [10, 20, 30], 0, 20, 24)
    x, w = hip.from_numpy(c["x"]), hip.from_numpy(c["w"])
    for offsets, held in (([0, 10, 1 << 40, 2**64 - 1], [(0, 10), (10, 60), None]), ([70, 80, 5, 9], [None, None, (5, 9)]),
                          ([20, 10, 10, 60], [None, None, (10, 60)])):
        off = hip.from_numpy(np.array(offsets, U64))
        yb = put(hip, np.full((60, 24), 9, np.float32))
        hip.dispatch("expert_linear_fwd", x=x, w=w, bias=None, y=yb[1], offsets=off, n_rows=60, n_experts=3, fan_in=20, fan_out=24,
                     relu=False)
        want = np.full((60, 24), 9.0)
        for e, s in enumerate(held):
            if s:
                want[s[0]:s[1]] = c["x"][s[0]:s[1]].astype(np.float64) @ c["w"][e].astype(np.float64).T
        got = get(hip, yb[0], 0, (60, 24))
        assert np.allclose(got, want, rtol=0, atol=23 * EPS * 20 * 16)  # |x w| below 16 each
        hip.mem_free(yb[0])


def test_no_rows(hip):
    w, off = hip.from_numpy(np.ones((2, 3, 4), np.float32)), hip.from_numpy(np.zeros(3, U64))
    gw, gb, one = hip.from_numpy(np.full((2, 3, 4), 5, np.float32)), hip.from_numpy(np.full((2, 3), 5, np.float32)), hip.from_numpy(np.zeros(1, np.float32))
    size = dict(n_rows=0, n_experts=2, fan_in=4, fan_out=3)
    hip.dispatch("expert_linear_fwd", x=one, w=w, bias=None, y=one, offsets=off, relu=False, **size)
    hip.dispatch("expert_linear_bwd", gy=one, x=one, w=w, act_in=None, gw=gw, gb=gb, gx=None, offsets=off, accumulate=True, **size)
    assert (hip.to_numpy(gw) == 5).all() and (hip.to_numpy(gb) == 5).all()
    hip.dispatch("expert_linear_bwd", gy=one, x=one, w=w, act_in=None, gw=gw, gb=gb, gx=None, offsets=off, accumulate=False, **size)
    assert (hip.to_numpy(gw) == 0).all() and (hip.to_numpy(gb) == 0).all()
