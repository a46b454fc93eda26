"""The operators built on the k largest of a row at sizes whose loads and stores pass by the memory-side cache: other instances of the
kernels than smaller inputs reach, at every row length where the kernels change."""
import numpy as np
import pytest

from test_gpu_distill import check, run
from topk_reference import NONE, expert_sort

pytestmark = pytest.mark.gpu
F32, U64 = np.float32, np.uint64
MI = 1 << 20


def rows_of(r, rows, cols, k):
    """Twelve different rows of a student and a teacher, each many times in a mixed order."""
    x = (r.standard_normal((12, cols)) * 2).astype(F32)
    indices = np.stack([r.permutation(cols)[:k] for _ in range(12)]).astype(U64)
    indices[3, 4] = indices[3, 1]   # one class twice
    indices[5, 2] = NONE            # padding
    teacher = -np.sort(-(r.standard_normal((12, k)) * 2).astype(F32), axis=1)
    which = r.integers(0, 12, rows)
    which[:2] = which[-2:] = 3, 5
    return x[which], teacher[which], indices[which]


def some_of(r, rows):
    return np.unique(np.concatenate([[0, 1, rows // 2, rows - 2, rows - 1], r.integers(0, rows, 20)]))


# columns: one for each kernel of the loss, of the gradient with it and of the gradient alone
@pytest.mark.parametrize("cols,k", [(300, 40), (1000, 40), (2000, 40), (2000, 65), (4001, 40), (8001, 40), (10001, 64), (32000, 64), (50257, 100),
                                    (60001, 20), (70001, 20)])
@pytest.mark.parametrize("way", ["apart", "fused", "fused, added", "apart, added"])
def test_distillation(hip, cols, k, way):
    add, fused = "added" in way, "fused" in way
    rows = 80 * MI // (cols * (2 if add and fused else 1)) + 3   # forward alone reads the logits, a gradient added to reads it as well
    r = np.random.default_rng(cols + k)
    x, teacher, indices = rows_of(r, rows, cols, k)
    w = np.ones(rows, F32)
    w[::7] = 0
    at = some_of(r, rows)
    grad0 = np.resize((r.standard_normal(1 * MI + 17)).astype(F32), x.shape) if add else None
    got = run(hip, x, teacher, indices, 2.0, w, grad0, fused)
    pick = {n: got[n][at] for n in ("stats", "row_loss", "grad")}
    # the scalar loss is held against the kernel's own row losses, all of them: rows / 64 + 16 halves of a step of each
    assert abs(got["loss"] - (w * got["row_loss"].astype(np.float64)).sum()) <= (rows / 64 + 16) * 2.0**-24 * np.abs(got["row_loss"]).astype(np.float64).sum()
    pick["loss"] = float((w[at] * pick["row_loss"].astype(np.float64)).sum())
    check(pick, x[at], teacher[at], indices[at], 2.0, w[at], grad0[at] if add else None)
    assert (got["row_loss"][::7] == 0).all()
    assert np.array_equal(got["grad"][::7], grad0[::7] if add else np.zeros_like(x[::7]))


# more than 64 Mi floats written; more than that read and written only; a narrow layer (16 lanes an entry), rows off the 16-byte grid
@pytest.mark.parametrize("tokens,k,width", [(65700, 8, 128), (66000, 9, 126), (8200, 8, 1030), (4200, 8, 1030), (33000, 8, 128), (8300, 64, 128)])
def test_rows_to_experts_and_back(hip, tokens, k, width):
    """Whole numbers and powers of two: every result is exact in any order of the sums."""
    n, n_experts = tokens * k, 64
    assert 2 * n * width + tokens * width > 64 * MI
    r = np.random.default_rng(tokens)
    experts = r.integers(0, n_experts + 1, n).astype(U64)    # the last: dropped
    _, slots = expert_sort(experts, n_experts)
    held = slots != NONE
    place = slots[held].astype(np.int64)
    token = np.arange(n)[held] // k
    x = r.integers(-4, 5, (tokens, width)).astype(F32)
    y = np.resize(r.integers(-4, 5, MI + 29).astype(F32), (n, width))
    w = (2.0 ** r.integers(-2, 2, n)).astype(F32)
    b = {"x": hip.from_numpy(x), "y": hip.from_numpy(y), "w": hip.from_numpy(w), "slots": hip.from_numpy(slots),
         "rows": hip.mem_alloc(F32, n * width), "out": hip.mem_alloc(F32, tokens * width), "w_g": hip.mem_alloc(F32, n)}
    size = dict(n_tokens=tokens, k=k, width=width)
    try:
        hip.mem_fill(b["rows"], 9.0)
        hip.dispatch("expert_dispatch", x=b["x"], slots=b["slots"], y=b["rows"], **size)
        rows = hip.to_numpy(b["rows"], (n, width))
        assert np.array_equal(rows[place], x[token]) and (rows[len(place):] == 9).all()

        def summed(weighted):
            out = np.zeros((tokens, width), F32)
            for j in range(k):   # in the order of j, all tokens at a time
                s = slots.reshape(tokens, k)[:, j]
                there = s != NONE
                term = y[s[there].astype(np.int64)]
                out[there] += term * w.reshape(tokens, k)[there, j, None] if weighted else term
            return out

        hip.dispatch("expert_combine", y=b["y"], slots=b["slots"], weights=b["w"], out=b["out"], **size)
        assert np.array_equal(hip.to_numpy(b["out"], (tokens, width)), summed(True))
        plain = summed(False)
        hip.dispatch("expert_dispatch_bwd", y_g=b["y"], slots=b["slots"], x_g=b["out"], accumulate=False, **size)
        assert np.array_equal(hip.to_numpy(b["out"], (tokens, width)), plain)
        hip.dispatch("expert_dispatch_bwd", y_g=b["y"], slots=b["slots"], x_g=b["out"], accumulate=True, **size)
        assert np.array_equal(hip.to_numpy(b["out"], (tokens, width)), 2 * plain)

        want_w = np.zeros(n, F32)
        want_w[held] = np.einsum("ij,ij->i", x[token], y[place])
        for want_rows, want_weights in ((True, True), (True, False), (False, True)):
            hip.mem_fill(b["rows"], 9.0)
            hip.mem_fill(b["w_g"], 9.0)
            hip.dispatch("expert_combine_bwd", out_g=b["x"], y=b["y"] if want_weights else None, slots=b["slots"], weights=b["w"],
                         y_g=b["rows"] if want_rows else None, weights_g=b["w_g"] if want_weights else None, **size)
            if want_rows:
                rows = hip.to_numpy(b["rows"], (n, width))
                assert np.array_equal(rows[place], x[token] * w[held][:, None]) and (rows[len(place):] == 9).all()
            assert (hip.to_numpy(b["w_g"]) == (want_w if want_weights else 9)).all()
    finally:
        for buf in b.values():
            hip.mem_free(buf)
