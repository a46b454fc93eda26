"""Argument checks of the operators built on the k largest of a row (include/zg_hip_topk.h), without a GPU: every refusal
happens on the host before any launch, so a context of zeros is all that the library reads on the way to one."""
import ctypes

import numpy as np
import pytest

from zigrad_amd._lib import TOPK_HEADER, Library, parse_header
from zigrad_amd.device import DevBuf, HipDevice

P = 1 << 20   # operands of the calls below lie at multiples of 1 MiB; nothing is read from them
A, B, C, D, E, F, G, H = (P * i for i in range(1, 9))
U64 = np.dtype(np.uint64)

# a call of each entry point that passes every check: {function: {parameter: value}}
GOOD = {
    "zg_hip_topk_fwd": dict(x=A, values=B, indices=C, rows=4, cols=16, k=3),
    "zg_hip_topk_bwd": dict(indices=A, y_g=B, x_g=C, rows=4, cols=16, k=3, accumulate=0),
    "zg_hip_distill_fwd": dict(logits=A, teacher=B, indices=C, row_weights=D, stats=E, row_loss=F, loss=G, rows=4, cols=16, k=3,
                               temperature=1.0),
    "zg_hip_distill_bwd": dict(logits=A, teacher=B, indices=C, row_weights=D, stats=E, grad=F, rows=4, cols=16, k=3,
                               temperature=1.0, accumulate=0),
    "zg_hip_distill_fwd_bwd": dict(logits=A, teacher=B, indices=C, row_weights=D, stats=E, row_loss=F, loss=G, grad=H, rows=4,
                                   cols=16, k=3, temperature=1.0, accumulate=0),
    "zg_hip_expert_sort": dict(experts=A, offsets=B, slots=C, n_entries=8, n_experts=4),
    "zg_hip_expert_dispatch": dict(x=A, slots=B, y=C, n_tokens=4, k=2, width=8),
    "zg_hip_expert_dispatch_bwd": dict(y_g=A, slots=B, x_g=C, n_tokens=4, k=2, width=8, accumulate=0),
    "zg_hip_expert_combine": dict(y=A, slots=B, weights=C, out=D, n_tokens=4, k=2, width=8),
    "zg_hip_expert_combine_bwd": dict(out_g=A, y=B, slots=C, weights=D, y_g=E, weights_g=F, n_tokens=4, k=2, width=8),
    "zg_hip_expert_linear_fwd": dict(x=A, w=B, bias=C, y=D, offsets=E, n_rows=4, n_experts=2, fan_in=8, fan_out=8, relu=0),
    "zg_hip_expert_linear_bwd": dict(gy=A, x=B, w=C, act_in=D, gw=E, gb=F, gx=G, offsets=H, n_rows=4, n_experts=2, fan_in=8,
                                     fan_out=8, accumulate=0),
}

# {function: [(changes to the call that passes, a word of the message)]}
BAD = {
    "zg_hip_topk_fwd": [(dict(k=0), "k = 0"), (dict(k=17), "k = 17"), (dict(cols=4096, k=513), "k = 513"), (dict(x=0), "null"),
                        (dict(values=0), "null"), (dict(indices=0), "null"), (dict(indices=C + 4), "8-byte"),
                        (dict(values=A + 4), "overlaps"), (dict(indices=A + 248), "overlaps"), (dict(indices=B), "overlaps"),
                        (dict(cols=1 << 33), "columns"), (dict(rows=1 << 60), "rows")],
    "zg_hip_topk_bwd": [(dict(k=0), "k = 0"), (dict(k=513), "k = 513"), (dict(x_g=0), "null"), (dict(y_g=0), "null"),
                        (dict(indices=0), "null"), (dict(indices=A + 4), "8-byte"), (dict(x_g=B), "overlaps"),
                        (dict(x_g=A + 92), "overlaps"), (dict(rows=1 << 60), "rows"), (dict(cols=1 << 33), "columns")],
    "zg_hip_distill_fwd": [(dict(rows=0), "empty"), (dict(cols=0), "empty"), (dict(k=0), "k = 0"), (dict(k=513), "k = 513"),
                           (dict(logits=0), "null"), (dict(teacher=0), "null"), (dict(indices=0), "null"), (dict(stats=0), "null"),
                           (dict(row_loss=0), "null"), (dict(loss=0), "null"), (dict(indices=C + 4), "8-byte"),
                           (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
                           (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
                           (dict(temperature=1e-45), "temperature"), (dict(temperature=9e-19), "temperature"),
                           (dict(temperature=1.1e18), "temperature"), (dict(stats=A), "overlaps"), (dict(row_loss=D), "overlaps"),
                           (dict(loss=F + 12), "overlap"), (dict(row_loss=E + 16), "overlap"), (dict(cols=1 << 33), "columns"),
                           (dict(rows=1 << 58), "rows")],
    "zg_hip_distill_bwd": [(dict(k=0), "k = 0"), (dict(stats=0), "null"), (dict(grad=0), "null"), (dict(grad=A), "overlaps"),
                           (dict(grad=E), "overlaps"), (dict(grad=D), "overlaps"), (dict(indices=C + 4), "8-byte"),
                           (dict(temperature=0.0), "temperature"), (dict(cols=1 << 33), "columns")],
    "zg_hip_distill_fwd_bwd": [(dict(rows=0), "empty"), (dict(grad=0), "null"), (dict(grad=A), "overlaps"), (dict(grad=G), "overlaps"),
                               (dict(grad=F), "overlaps"), (dict(stats=0), "null"), (dict(k=0), "k = 0")],
    "zg_hip_expert_sort": [(dict(n_experts=0), "experts"), (dict(n_experts=1025), "experts"), (dict(n_entries=1 << 32), "entries"),
                           (dict(experts=0), "null"), (dict(offsets=0), "null"), (dict(slots=0), "null"), (dict(slots=C + 4), "8-byte"),
                           (dict(offsets=B + 4), "8-byte"), (dict(experts=A + 4), "8-byte"), (dict(slots=A + 8), "overlap"),
                           (dict(offsets=A), "overlap"), (dict(offsets=C), "overlap")],
    "zg_hip_expert_dispatch": [(dict(k=0), "k = 0"), (dict(k=65), "k = 65"), (dict(x=0), "null"), (dict(slots=0), "null"),
                               (dict(y=0), "null"), (dict(y=A), "overlaps"), (dict(y=B), "overlaps"), (dict(slots=B + 4), "8-byte"),
                               (dict(n_tokens=1 << 40, width=1 << 30), "rows")],
    "zg_hip_expert_dispatch_bwd": [(dict(k=0), "k = 0"), (dict(y_g=0), "null"), (dict(x_g=0), "null"), (dict(slots=0), "null"),
                                   (dict(x_g=A), "overlaps"), (dict(x_g=B), "overlaps"), (dict(slots=B + 4), "8-byte")],
    "zg_hip_expert_combine": [(dict(k=65), "k = 65"), (dict(y=0), "null"), (dict(weights=0), "null"), (dict(out=0), "null"),
                              (dict(out=A), "overlaps"), (dict(out=C), "overlaps"), (dict(slots=B + 4), "8-byte")],
    "zg_hip_expert_combine_bwd": [(dict(k=0), "k = 0"), (dict(out_g=0), "null"), (dict(slots=0), "null"), (dict(weights=0), "null"),
                                  (dict(y=0), "null"), (dict(y_g=B), "overlaps"), (dict(y_g=A), "overlaps"),
                                  (dict(weights_g=D), "overlaps"), (dict(weights_g=E), "overlaps"), (dict(weights_g=A), "overlaps")],
    "zg_hip_expert_linear_fwd": [(dict(n_experts=0), "experts"), (dict(n_experts=1025), "experts"), (dict(n_rows=1 << 31), "rows"),
                                 (dict(fan_in=0), "no inputs"), (dict(fan_in=1 << 21), "layer"), (dict(fan_out=1 << 21), "layer"),
                                 (dict(x=0), "null"), (dict(w=0), "null"), (dict(y=0), "null"), (dict(offsets=0), "offsets"),
                                 (dict(offsets=E + 4), "8-byte"), (dict(y=A), "overlaps"), (dict(y=B), "overlaps"),
                                 (dict(y=C), "overlaps")],
    "zg_hip_expert_linear_bwd": [(dict(gy=0), "null"), (dict(x=0), "null"), (dict(w=0), "null"), (dict(gw=0), "null"),
                                 (dict(offsets=0), "offsets"), (dict(gw=C), "overlaps"), (dict(gx=A), "overlaps"),
                                 (dict(gx=D), "overlaps"), (dict(gb=E), "overlap"), (dict(gx=E), "overlap"),
                                 (dict(fan_in=1 << 21), "layer"), (dict(n_rows=1 << 31), "rows"), (dict(n_experts=0), "experts")],
}

# calls with nothing to do: accepted, nothing is launched
NOTHING = {
    "zg_hip_topk_fwd": [dict(rows=0)],
    "zg_hip_topk_bwd": [dict(rows=0), dict(cols=0)],
    "zg_hip_distill_bwd": [dict(rows=0), dict(cols=0)],
    "zg_hip_expert_dispatch": [dict(n_tokens=0), dict(width=0)],
    "zg_hip_expert_dispatch_bwd": [dict(n_tokens=0), dict(width=0)],
    "zg_hip_expert_combine": [dict(n_tokens=0), dict(width=0)],
    "zg_hip_expert_combine_bwd": [dict(n_tokens=0), dict(y_g=0, weights_g=0, width=0)],
    "zg_hip_expert_linear_fwd": [dict(n_rows=0), dict(fan_out=0)],
    "zg_hip_expert_linear_bwd": [dict(fan_out=0), dict(fan_in=0)],
}


@pytest.fixture(scope="module")
def library():
    return Library()


def call(library, name, changes):
    zeros = (ctypes.c_char * (1 << 20))()
    p = {**GOOD[name], **changes}
    names = [n for n, _ in library.protos[name][1]]
    assert names[0] == "ctx" and set(names[1:]) == set(p), name
    rc = getattr(library.cdll, name)(ctypes.addressof(zeros), *[p[n] for n in names[1:]])
    return rc, library.last_error()


@pytest.mark.parametrize("name,changes,word", [(n, c, w) for n, rows in BAD.items() for c, w in rows])
def test_bad_arguments_are_refused_before_any_launch(library, name, changes, word):
    rc, message = call(library, name, changes)
    assert rc == 1 and word in message, (rc, message)


@pytest.mark.parametrize("name,changes", [(n, c) for n, rows in NOTHING.items() for c in rows])
def test_calls_with_nothing_to_do_succeed(library, name, changes):
    assert call(library, name, changes)[0] == 0


def test_every_entry_point_of_the_header_is_checked_and_refuses_a_null_context(library):
    declared = parse_header(TOPK_HEADER)
    assert set(declared) == set(GOOD) == set(BAD)
    for name in declared:
        args = [GOOD[name][n] for n, _ in library.protos[name][1][1:]]
        assert getattr(library.cdll, name)(None, *args) == 1
        assert "null context" in library.last_error()


def _device():
    dev = HipDevice.__new__(HipDevice)
    dev._ctx = None

    def call(name, *args):
        raise AssertionError("the library was called")

    dev._call = call
    return dev


@pytest.mark.parametrize("name,kind,short", [
    ("topk_fwd", dict(x=64, values=12, indices=12), "x"), ("topk_fwd", dict(x=64, values=12, indices=12), "indices"),
    ("topk_bwd", dict(indices=12, y_g=12, x_g=64), "x_g"),
    ("distill_fwd", dict(logits=64, teacher=12, indices=12, stats=8, row_loss=4, loss=1, weights=4), "stats"),
    ("distill_fwd", dict(logits=64, teacher=12, indices=12, stats=8, row_loss=4, loss=1, weights=4), "weights"),
    ("distill_bwd", dict(logits=64, teacher=12, indices=12, stats=8, grad=64), "grad"),
    ("distill_fwd_bwd", dict(logits=64, teacher=12, indices=12, stats=8, row_loss=4, loss=1, grad=64), "loss")])
def test_short_buffers_and_wrong_types_are_refused_by_the_device(name, kind, short):
    index = {"indices"}
    bufs = {n: DevBuf(P * (i + 1), size, U64 if n in index else np.dtype(np.float32)) for i, (n, size) in enumerate(kind.items())}
    size = dict(rows=4, cols=16, k=3)
    with pytest.raises(AssertionError, match="the library was called"):
        _device().dispatch(name, **bufs, **size)
    less = DevBuf(bufs[short].ptr, bufs[short].n - 1, bufs[short].dtype)
    with pytest.raises(ValueError, match=short):
        _device().dispatch(name, **{**bufs, short: less}, **size)
    other = DevBuf(bufs[short].ptr, bufs[short].n, np.dtype(np.float32) if short in index else U64)
    with pytest.raises(TypeError, match=short):
        _device().dispatch(name, **{**bufs, short: other}, **size)


@pytest.mark.parametrize("name,kind,short,size", [
    ("expert_sort", dict(experts=8, offsets=5, slots=8), "offsets", dict(n_experts=4)),
    ("expert_sort", dict(experts=8, offsets=5, slots=8), "slots", dict(n_experts=4)),
    ("expert_dispatch", dict(x=32, slots=8, y=64), "y", dict(n_tokens=4, k=2, width=8)),
    ("expert_dispatch_bwd", dict(y_g=64, slots=8, x_g=32), "x_g", dict(n_tokens=4, k=2, width=8)),
    ("expert_combine", dict(y=64, slots=8, weights=8, out=32), "weights", dict(n_tokens=4, k=2, width=8)),
    ("expert_combine_bwd", dict(out_g=32, slots=8, weights=8, y=64, y_g=64, weights_g=8), "weights_g", dict(n_tokens=4, k=2, width=8)),
    ("expert_linear_fwd", dict(x=32, w=128, bias=16, y=32, offsets=3), "bias",
     dict(n_rows=4, n_experts=2, fan_in=8, fan_out=8, relu=False)),
    ("expert_linear_bwd", dict(gy=32, x=32, w=128, act_in=32, gw=128, gb=16, gx=32, offsets=3), "gw",
     dict(n_rows=4, n_experts=2, fan_in=8, fan_out=8))])
def test_short_expert_buffers_are_refused_by_the_device(name, kind, short, size):
    index = {"experts", "offsets", "slots"}
    bufs = {n: DevBuf(P * (i + 1), n_el, U64 if n in index else np.dtype(np.float32)) for i, (n, n_el) in enumerate(kind.items())}
    with pytest.raises(AssertionError, match="the library was called"):
        _device().dispatch(name, **bufs, **size)
    less = DevBuf(bufs[short].ptr, bufs[short].n - 1, bufs[short].dtype)
    with pytest.raises(ValueError, match=short):
        _device().dispatch(name, **{**bufs, short: less}, **size)
