"""The operators built on the k largest of a row together, as a training step of a layer of experts taught by a larger model uses
them: against the same step in 64 bits, recorded and replayed, beside work that waits in the context, and in two contexts at
once."""
import numpy as np
import pytest

from conftest import rel_fro
from topk_reference import distill, expert_sort
from zigrad_amd import HipDevice
from zigrad_amd._lib import TOPK_HEADER, parse_header

pytestmark = pytest.mark.gpu
U64 = np.uint64
F32 = np.float32


class Step:
    """Router, k of E experts with one hidden layer each, logits, loss against the teacher's t best, and every gradient."""

    def __init__(self, tokens=70, width=24, hidden=40, classes=33, experts=6, k=2, kept=5, temp=2.0, seed=0):
        self.__dict__.update(tokens=tokens, width=width, hidden=hidden, classes=classes, experts=experts, k=k, kept=kept, temp=temp)
        r = np.random.default_rng(seed)
        # multiples of 1/8 below 8: the router's products and sums are exact, so both precisions choose the same experts
        self.x = (r.integers(-16, 17, (tokens, width)) / 8).astype(F32)
        self.params = {"router": (r.integers(-16, 17, (experts, width)) / 8).astype(F32),
                       "w1": (r.standard_normal((experts, hidden, width)) * np.sqrt(2 / width)).astype(F32),
                       "b1": (r.standard_normal((experts, hidden)) * 0.1).astype(F32),
                       "w2": (r.standard_normal((experts, classes, hidden)) * np.sqrt(2 / hidden)).astype(F32),
                       "b2": (r.standard_normal((experts, classes)) * 0.1).astype(F32)}
        self.teacher = (r.standard_normal((tokens, classes)) * 2).astype(F32)

    # the step in 64 bits
    def reference(self, params=None, x=None):
        p = {n: v.astype(np.float64) for n, v in (params or self.params).items()}
        x = (self.x if x is None else x).astype(np.float64)
        best = lambda a, k: np.argsort(-a, axis=1, kind="stable")[:, :k]  # noqa: E731
        scores = x @ p["router"].T
        chosen = best(scores, self.k)
        values = np.take_along_axis(scores, chosen, axis=1)
        gates = np.exp(values - values.max(axis=1, keepdims=True))
        gates /= gates.sum(axis=1, keepdims=True)
        hid = np.stack([[np.maximum(p["w1"][e] @ x[t] + p["b1"][e], 0) for e in chosen[t]] for t in range(self.tokens)])
        outs = np.stack([[p["w2"][e] @ hid[t, j] + p["b2"][e] for j, e in enumerate(chosen[t])] for t in range(self.tokens)])
        logits = (gates[:, :, None] * outs).sum(axis=1)
        kept = best(self.teacher.astype(np.float64), self.kept)
        ref = distill(logits, np.take_along_axis(self.teacher, kept, axis=1), kept.astype(U64), self.temp)
        g = {n: np.zeros_like(v) for n, v in p.items()}
        g["x"] = np.zeros_like(x)
        for t in range(self.tokens):
            lg = ref["grad"][t]
            gate_g = outs[t] @ lg
            value_g = gates[t] * (gate_g - (gates[t] * gate_g).sum())
            for j, e in enumerate(chosen[t]):
                og = gates[t, j] * lg
                g["w2"][e] += np.outer(og, hid[t, j])
                g["b2"][e] += og
                hg = (p["w2"][e].T @ og) * (hid[t, j] > 0)
                g["w1"][e] += np.outer(hg, x[t])
                g["b1"][e] += hg
                g["x"][t] += p["w1"][e].T @ hg + value_g[j] * p["router"][e]
                g["router"][e] += value_g[j] * x[t]
        return ref["loss"], g

    # the same through the library
    def upload(self, hip):
        self.hip = hip
        n, t = self.tokens * self.k, self.tokens
        b = self.b = {"x": hip.from_numpy(self.x), "teacher": hip.from_numpy(self.teacher)}
        for name, v in self.params.items():
            b[name], b[name + "_g"] = hip.from_numpy(v), hip.mem_alloc(F32, v.size)
        for name, size in (("scores", t * self.experts), ("values", t * self.k), ("gates", t * self.k), ("rows", n * self.width),
                           ("hid", n * self.hidden), ("outs", n * self.classes), ("logits", t * self.classes),
                           ("kept_v", t * self.kept), ("stats", 2 * t), ("row_loss", t), ("loss", 1), ("logits_g", t * self.classes),
                           ("outs_g", n * self.classes), ("gates_g", t * self.k), ("hid_g", n * self.hidden), ("rows_g", n * self.width),
                           ("values_g", t * self.k), ("scores_g", t * self.experts), ("x_g", t * self.width)):
            b[name] = hip.from_numpy(np.zeros(size, F32))
        for name, size in (("chosen", n), ("kept", t * self.kept), ("offsets", self.experts + 1), ("slots", n)):
            b[name] = hip.from_numpy(np.zeros(size, U64))

    def run(self):
        hip, b, t = self.hip, self.b, self.tokens
        d = hip.dispatch
        place = dict(n_tokens=t, k=self.k)
        e1 = dict(offsets=b["offsets"], n_rows=t * self.k, n_experts=self.experts, fan_in=self.width, fan_out=self.hidden)
        e2 = dict(e1, fan_in=self.hidden, fan_out=self.classes)
        d("linear_fwd", x=b["x"], w=b["router"], bias=None, y=b["scores"], batch=t, fan_in=self.width, fan_out=self.experts, relu=False)
        d("topk_fwd", x=b["scores"], values=b["values"], indices=b["chosen"], rows=t, cols=self.experts, k=self.k)
        d("softmax_fwd", x=b["values"], y=b["gates"], rows=t, cols=self.k)
        d("expert_sort", experts=b["chosen"], offsets=b["offsets"], slots=b["slots"], n_experts=self.experts)
        d("expert_dispatch", x=b["x"], slots=b["slots"], y=b["rows"], width=self.width, **place)
        d("expert_linear_fwd", x=b["rows"], w=b["w1"], bias=b["b1"], y=b["hid"], relu=True, **e1)
        d("expert_linear_fwd", x=b["hid"], w=b["w2"], bias=b["b2"], y=b["outs"], relu=False, **e2)
        d("expert_combine", y=b["outs"], slots=b["slots"], weights=b["gates"], out=b["logits"], width=self.classes, **place)
        d("topk_fwd", x=b["teacher"], values=b["kept_v"], indices=b["kept"], rows=t, cols=self.classes, k=self.kept)
        loss = dict(logits=b["logits"], teacher=b["kept_v"], indices=b["kept"], stats=b["stats"], rows=t, cols=self.classes, k=self.kept,
                    temperature=self.temp)
        d("distill_fwd", row_loss=b["row_loss"], loss=b["loss"], **loss)
        d("distill_bwd", grad=b["logits_g"], accumulate=False, **loss)
        d("expert_combine_bwd", out_g=b["logits_g"], y=b["outs"], slots=b["slots"], weights=b["gates"], y_g=b["outs_g"],
          weights_g=b["gates_g"], width=self.classes, **place)
        d("expert_linear_bwd", gy=b["outs_g"], x=b["hid"], w=b["w2"], act_in=b["hid"], gw=b["w2_g"], gb=b["b2_g"], gx=b["hid_g"],
          accumulate=False, **e2)
        d("expert_linear_bwd", gy=b["hid_g"], x=b["rows"], w=b["w1"], act_in=None, gw=b["w1_g"], gb=b["b1_g"], gx=b["rows_g"],
          accumulate=False, **e1)
        d("expert_dispatch_bwd", y_g=b["rows_g"], slots=b["slots"], x_g=b["x_g"], width=self.width, accumulate=False, **place)
        hip.mem_fill(b["values_g"], 0.0)
        d("softmax_bwd", y=b["gates"], y_g=b["gates_g"], x_g=b["values_g"], rows=t, cols=self.k)
        d("topk_bwd", indices=b["chosen"], y_g=b["values_g"], x_g=b["scores_g"], rows=t, cols=self.experts, k=self.k, accumulate=False)
        hip.mem_fill(b["router_g"], 0.0)
        d("matmul", A=b["scores_g"], B=b["x"], C=b["router_g"], m=self.experts, n=self.width, k=t, trans_a=True, trans_b=False,
          lda=self.experts, ldb=self.width, ldc=self.width, alpha=1.0, beta=1.0)
        d("matmul", A=b["scores_g"], B=b["router"], C=b["x_g"], m=t, n=self.width, k=self.experts, trans_a=False, trans_b=False,
          lda=self.experts, ldb=self.width, ldc=self.width, alpha=1.0, beta=1.0)

    def results(self):
        names = ["loss", "x_g"] + [n + "_g" for n in self.params]
        return {n: self.hip.to_numpy(self.b[n]) for n in names}

    def free(self):
        for buf in self.b.values():
            self.hip.mem_free(buf)


@pytest.mark.parametrize("sizes", [{}, dict(tokens=1, experts=1, k=1), dict(tokens=300, width=96, hidden=64, classes=100, experts=16, k=4, kept=20),
                                   dict(tokens=33, width=7, hidden=5, classes=9, experts=8, k=8, kept=9)])
def test_a_training_step_against_64_bits(hip, sizes):
    """Dot products of at most 300 terms over eight products one behind the other: 8 * 302 halves of a step, 1.5e-4, if every
    rounding went the same way; they do not, and the norm over many elements is held to a third of it."""
    s = Step(**sizes)
    loss, grads = s.reference()
    s.upload(hip)
    s.run()
    got = s.results()
    s.free()
    assert abs(got["loss"][0] - loss) <= 5e-5 * max(1.0, abs(loss))
    for name, want in grads.items():
        if np.linalg.norm(want) > 1e-12:
            assert rel_fro(got[name + "_g"], want) <= 5e-5, name


def test_the_step_in_64_bits_is_the_gradient_that_differences_say():
    """Central differences of step 1e-5 away from kinks and changes of choice: off by about h^2 and by rounding over h."""
    s = Step(tokens=5, width=6, hidden=7, classes=8, experts=4, k=2, kept=3, seed=11)
    r = np.random.default_rng(2)
    s.x = r.standard_normal(s.x.shape)
    s.params = {n: r.standard_normal(v.shape) for n, v in s.params.items()}
    _, grads = s.reference()
    h = 1e-5
    for name in (*s.params, "x"):
        for _ in range(6):
            at = tuple(r.integers(0, d) for d in (s.x if name == "x" else s.params[name]).shape)
            moved = []
            for sign in (h, -h):
                p, x = {n: v.copy() for n, v in s.params.items()}, s.x.copy()
                (x if name == "x" else p[name])[at] += sign
                moved.append(s.reference(p, x)[0])
            assert abs((moved[0] - moved[1]) / (2 * h) - grads[name][at]) <= 1e-7 * max(1.0, abs(grads[name][at])), (name, at)


def test_a_recorded_step_replays_what_eager_calls_leave(hip):
    """New inputs before every replay, eager work and waits in between; the recording's results equal the eager ones bit for bit."""
    s = Step(tokens=200, width=64, hidden=48, classes=120, experts=16, k=4, kept=12)
    s.upload(hip)
    r = np.random.default_rng(5)
    batches = [(r.integers(-16, 17, s.x.shape) / 8).astype(F32) for _ in range(4)]
    eager = []
    for x in batches:
        hip.mem_transfer(x, s.b["x"], "HtoD")
        s.run()
        eager.append(s.results())
    hip.sync()
    hip.graph_open()
    try:
        s.run()
    finally:
        graph = hip.graph_save()
    for k in (0, 1, 2, 3, 1):
        hip.mem_transfer(batches[k], s.b["x"], "HtoD")
        hip.mem_fill(s.b["loss"], -1.0)
        graph.run()
        got = s.results()
        for name, want in eager[k].items():
            assert np.array_equal(got[name], want), (k, name)
        other = hip.from_numpy(np.ones(1000, F32))
        hip.dispatch("scale", x=other, alpha=2.0)
        hip.sync()
        hip.mem_free(other)
    graph.free()
    s.free()


@pytest.mark.parametrize("op", ["topk_fwd", "expert_sort", "expert_linear_bwd"])
def test_a_recording_without_a_run_before_it(hip, op):
    """A call that would have to allocate its workspace is refused in a recording; the context and the recording go on."""
    dev = HipDevice(0)  # no workspace yet
    try:
        if op == "topk_fwd":
            x = np.random.default_rng(1).standard_normal((2, 40000)).astype(F32)
            b = dict(x=dev.from_numpy(x), values=dev.mem_alloc(F32, 16), indices=dev.mem_alloc(U64, 16))
            size = dict(rows=2, cols=40000, k=8)
        elif op == "expert_sort":
            experts = np.random.default_rng(1).integers(0, 9, 5000).astype(U64)
            b = dict(experts=dev.from_numpy(experts), offsets=dev.mem_alloc(U64, 10), slots=dev.mem_alloc(U64, 5000))
            size = dict(n_experts=9)
        else:
            b = dict(offsets=dev.from_numpy((np.arange(71) * 12).astype(U64)), gb=dev.mem_alloc(F32, 70 * 8), w=None, act_in=None, gx=None,
                     **{n: dev.from_numpy(np.ones(840 * 8, F32)) for n in ("gy", "x")}, gw=dev.mem_alloc(F32, 70 * 64))
            size = dict(n_rows=840, n_experts=70, fan_in=8, fan_out=8, accumulate=False)
        other = dev.from_numpy(np.ones(4, F32))
        dev.sync()
        dev.graph_open()
        try:
            with pytest.raises(RuntimeError):
                dev.dispatch(op, **b, **size)
            dev.dispatch("scale", x=other, alpha=2.0)
        finally:
            graph = dev.graph_save()
        graph.run()
        graph.run()
        assert (dev.to_numpy(other) == 4).all()
        dev.dispatch(op, **b, **size)  # eagerly: the workspace is there now
        graph.free()
        dev.sync()
        dev.graph_open()
        try:
            dev.dispatch(op, **b, **size)
        finally:
            graph = dev.graph_save()
        out = {"topk_fwd": "indices", "expert_sort": "slots", "expert_linear_bwd": "gw"}[op]
        want = dev.to_numpy(b[out])
        for _ in range(2):
            dev.mem_fill(b[out], 77)
            graph.run()
            assert np.array_equal(dev.to_numpy(b[out]), want)
        if op == "expert_linear_bwd":
            assert (want == 12).all()
        graph.free()
    finally:
        dev.deinit()


def test_two_contexts_at_once(hip):
    """Each context orders and multiplies on its own stream with its own workspace."""
    steps = [Step(tokens=3000, width=40, hidden=56, classes=65, experts=32, k=4, kept=8, seed=7), None]
    other = HipDevice(0)
    try:
        alone = []
        steps[0].upload(hip)
        steps[0].run()
        alone = steps[0].results()
        steps[1] = Step(tokens=3000, width=40, hidden=56, classes=65, experts=32, k=4, kept=8, seed=7)
        steps[1].upload(other)
        other.sync()
        for _ in range(3):
            steps[0].run()
            steps[1].run()
        for s in steps:
            got = s.results()
            assert all(np.array_equal(got[n], alone[n]) for n in alone)
            s.free()
    finally:
        other.deinit()


# ---- beside work that waits in the context -------------------------------------------------------------------
def _ops():
    """{op: (float inputs, index inputs, outputs, sizes)}: one call of each."""
    r = np.random.default_rng(8)
    f = lambda *s: r.standard_normal(s).astype(F32)  # noqa: E731
    experts = r.integers(0, 5, 40).astype(U64)
    offsets, slots = expert_sort(experts, 4)
    chosen = np.stack([r.permutation(30)[:4] for _ in range(20)]).astype(U64)
    held = int(offsets[-1])
    loss = dict(rows=20, cols=30, k=4, temperature=2.0)
    place = dict(n_tokens=20, k=2, width=12)
    layer = dict(n_rows=40, n_experts=4, fan_in=12, fan_out=9)
    assert held < 40
    return {
        "topk_fwd": (dict(x=f(20, 30)), {}, dict(values=80, indices=(80,)), dict(rows=20, cols=30, k=4)),
        "topk_bwd": (dict(y_g=f(20, 4)), dict(indices=chosen), dict(x_g=600), dict(rows=20, cols=30, k=4)),
        "distill_fwd": (dict(logits=f(20, 30), teacher=f(20, 4)), dict(indices=chosen), dict(stats=40, row_loss=20, loss=1), loss),
        "distill_bwd": (dict(logits=f(20, 30), teacher=f(20, 4), stats=np.abs(f(20, 2))), dict(indices=chosen), dict(grad=600), loss),
        "distill_fwd_bwd": (dict(logits=f(20, 30), teacher=f(20, 4), weights=f(20)), dict(indices=chosen),
                            dict(stats=40, row_loss=20, loss=1, grad=600), loss),
        "expert_sort": ({}, dict(experts=experts), dict(offsets=(5,), slots=(40,)), dict(n_experts=4)),
        "expert_dispatch": (dict(x=f(20, 12)), dict(slots=slots), dict(y=480), place),
        "expert_dispatch_bwd": (dict(y_g=f(40, 12)), dict(slots=slots), dict(x_g=240), place),
        "expert_combine": (dict(y=f(40, 12), weights=f(40)), dict(slots=slots), dict(out=240), place),
        "expert_combine_bwd": (dict(out_g=f(20, 12), y=f(40, 12), weights=f(40)), dict(slots=slots), dict(y_g=480, weights_g=40), place),
        "expert_linear_fwd": (dict(x=f(40, 12), w=f(4, 9, 12), bias=f(4, 9)), dict(offsets=offsets), dict(y=360), dict(layer, relu=True)),
        "expert_linear_bwd": (dict(gy=f(40, 9), x=f(40, 12), w=f(4, 9, 12), act_in=f(40, 12)), dict(offsets=offsets),
                              dict(gw=432, gb=36, gx=480), layer),
    }


def _beside_waiting_work(hip, op, wait):
    """The op's inputs come out of small elementwise ops, its outputs are filled before and scaled after: all calls that wait in the
    context for the next one.  wait: each is waited for instead."""
    floats, indices, outputs, sizes = _ops()[op]
    pause = hip.sync if wait else (lambda: None)
    ins = {n: hip.from_numpy(v) for n, v in {**floats, **indices}.items()}
    outs = {n: hip.mem_alloc(U64 if isinstance(s, tuple) else F32, s[0] if isinstance(s, tuple) else s) for n, s in outputs.items()}
    hip.sync()
    for n in floats:
        hip.dispatch("mul", x=ins[n], y=1.5, z=ins[n])
        pause()
    for n, b in outs.items():
        hip.mem_fill(b, 3 if b.dtype == U64 else 0.25)
        pause()
    hip.dispatch(op, **ins, **outs, **sizes)
    pause()
    for b in outs.values():
        if b.dtype == np.dtype(F32):
            hip.dispatch("mul", x=b, y=2.0, z=b)
            pause()
    got = {n: hip.to_numpy(b) for n, b in outs.items()}
    for b in (*ins.values(), *outs.values()):
        hip.mem_free(b)
    return got


@pytest.mark.parametrize("op", sorted(_ops()))
def test_beside_work_that_waits(hip, op):
    lazy, want = _beside_waiting_work(hip, op, False), _beside_waiting_work(hip, op, True)
    for n in want:
        assert np.array_equal(lazy[n], want[n]), n


def test_every_entry_point_of_the_header_is_run_beside_waiting_work():
    assert {"zg_hip_" + op for op in _ops()} == set(parse_header(TOPK_HEADER))
