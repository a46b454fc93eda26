"""Cases for the operators built on the k largest of a row: selection (`topk`), distillation from a teacher's top logits
(`distill`), rows routed to experts and back (`experts`) and the experts' Linear products (`expert_linear`).

Values are fp32 and indices 64-bit, as everywhere in this library.  `run` computes a case either in plain torch
operations or, with `own` set, through `HipDevice.dispatch`.
"""
import math

import numpy as np
import torch

own = False

_DROPPED = -1  # slot of an entry that goes to no expert: the largest 64-bit index


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the router of a small expert layer: one short row per token of a batch of 64
        {"name": "topk router b64", "op": "topk", "dir": "fwd", "rows": 64, "cols": 64, "k": 2},
        # keeping a teacher's 64 best logits for a pass of a large-vocabulary classifier
        {"name": "topk teacher 8192x32000", "op": "topk", "dir": "fwd", "rows": 8192, "cols": 32000, "k": 64},
        # the router's gradient in a training step: eight chosen experts of 256 per token, odd number of tokens
        {"name": "topk bwd 16383x256", "op": "topk", "dir": "bwd", "rows": 16383, "cols": 256, "k": 8, "acc": False},
        # the batch-64 ten-class classifier taught by the three best logits of a larger one
        {"name": "distill step 64x10", "op": "distill", "dir": "fwd_bwd", "rows": 64, "cols": 10, "k": 3, "temp": 2.0,
         "weights": False, "acc": False},
        # evaluation of the loss over a large vocabulary, some rows padding
        {"name": "distill fwd 8192x32000", "op": "distill", "dir": "fwd", "rows": 8192, "cols": 32000, "k": 64, "temp": 2.0,
         "weights": True, "acc": False},
        # a training step over rows off the 16-byte grid
        {"name": "distill step 2048x50257", "op": "distill", "dir": "fwd_bwd", "rows": 2048, "cols": 50257, "k": 100,
         "temp": 1.0, "weights": True, "acc": False},
        # serving a few tokens: order them by expert, lay their rows out
        {"name": "experts dispatch 16", "op": "experts", "dir": "dispatch", "tokens": 16, "k": 2, "experts": 8, "width": 1024},
        # rows back to their tokens in evaluation, odd number of tokens and a width off the 16-byte grid
        {"name": "experts combine 4095", "op": "experts", "dir": "combine", "tokens": 4095, "k": 6, "experts": 64, "width": 1030},
        # there and back in a training step, forward and backward
        {"name": "experts train 8192", "op": "experts", "dir": "train", "tokens": 8192, "k": 8, "experts": 64, "width": 1024},
        # the products of a few served tokens: bounded by reading the weights
        {"name": "expert linear fwd 32", "op": "expert_linear", "dir": "fwd", "rows": 32, "experts": 8, "fan_in": 1024,
         "fan_out": 2048, "bias": True, "relu": True},
        # evaluation with ragged groups and odd layer sizes
        {"name": "expert linear fwd 8190", "op": "expert_linear", "dir": "fwd", "rows": 8190, "experts": 32, "fan_in": 1000,
         "fan_out": 1030, "bias": True, "relu": False},
        # the backward pass of a training step
        {"name": "expert linear bwd 16384", "op": "expert_linear", "dir": "bwd", "rows": 16384, "experts": 16, "fan_in": 1024,
         "fan_out": 2048, "bias": True, "relu": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["topk", "distill", "experts", "expert_linear"])
    if op in ("topk", "distill"):
        cols = _log_int(rng, 8 if op == "topk" else 10, 128001)
        rows = _log_int(rng, 1, min(65536, 8192 * 32000 // cols))
        k = _log_int(rng, 1, min(cols, 128))
        if op == "topk":
            way = rng.choice(["fwd", "fwd", "bwd"])
            if way == "fwd":
                return {"op": op, "dir": way, "rows": rows, "cols": cols, "k": k}
            return {"op": op, "dir": way, "rows": rows, "cols": cols, "k": k, "acc": rng.random() < 0.5}
        return {"op": op, "dir": rng.choice(["fwd", "bwd", "fwd_bwd"]), "rows": rows, "cols": cols, "k": k,
                "temp": rng.choice([0.5, 1.0, 2.0, 4.0]), "weights": rng.random() < 0.5, "acc": rng.random() < 0.5}
    if op == "experts":
        k = rng.randint(1, 8)
        experts = _log_int(rng, k, 256)
        width = _log_int(rng, 16, 4096)
        tokens = _log_int(rng, 1, max(1, min(32768, 8192 * 8 * 1024 // (k * width))))
        return {"op": op, "dir": rng.choice(["dispatch", "combine", "train"]), "tokens": tokens, "k": k, "experts": experts,
                "width": width}
    experts = _log_int(rng, 1, 64)
    fan_in, fan_out = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
    while experts * fan_in * fan_out > 128 << 20:
        experts = (experts + 1) // 2
    rows = _log_int(rng, 1, max(1, min(16384, 16384 * 1024 * 2048 // (fan_in * fan_out))))
    return {"op": op, "dir": rng.choice(["fwd", "bwd"]), "rows": rows, "experts": experts, "fan_in": fan_in, "fan_out": fan_out,
            "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}


def work(case):
    if case["op"] == "topk":
        r, c, k = case["rows"], case["cols"], case["k"]
        if case["dir"] == "fwd":
            return {"bytes": 4 * r * c + 12 * r * k, "flops": 0}
        # accumulating touches the chosen places only; else every place is written
        return {"bytes": 12 * r * k + (8 * r * k if case["acc"] else 4 * r * c), "flops": 0}
    if case["op"] == "distill":
        r, c, k = case["rows"], case["cols"], case["k"]
        real = r * 15 // 16 if case["weights"] else r  # rows that are no padding: only their logits are needed
        read = 4 * real * c + 12 * real * k + (4 * r if case["weights"] else 0)
        if case["dir"] == "fwd":
            return {"bytes": read + 12 * r + 4, "flops": 4 * r * c}
        grad = 4 * r * c * (2 if case["acc"] else 1)
        if case["dir"] == "bwd":
            return {"bytes": read + 8 * r + grad, "flops": 5 * r * c}
        return {"bytes": read + 12 * r + 4 + grad, "flops": 9 * r * c}
    if case["op"] == "experts":
        t, k, e, d = case["tokens"], case["k"], case["experts"], case["width"]
        n = t * k
        sort, there, back = 16 * n + 8 * (e + 1), 4 * t * d + 4 * n * d + 8 * n, 4 * n * d + 12 * n + 4 * t * d
        if case["dir"] == "dispatch":
            return {"bytes": sort + there, "flops": 0}
        if case["dir"] == "combine":
            return {"bytes": back, "flops": 2 * n * d}
        return {"bytes": sort + there + back + (4 * t * d + 8 * n * d + 16 * n) + (4 * n * d + 8 * n + 4 * t * d),
                "flops": 6 * n * d}
    n, e, i, o = case["rows"], case["experts"], case["fan_in"], case["fan_out"]
    used = min(n, e) * i * o  # weights of experts that have rows, at most
    bias = e * o if case["bias"] else 0
    if case["dir"] == "fwd":
        return {"bytes": 4 * (n * i + n * o + used + bias), "flops": 2 * n * i * o}
    # gy, x (the gate is the same array) and w are read; gx and the gradients of all weights and biases are written
    return {"bytes": 4 * (n * o + n * i + used + n * i + e * i * o + bias), "flops": 4 * n * i * o}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda").mul_(scale)


def _empty(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def _choices(g, tokens, k, experts):
    """k different experts per token, some experts far more popular than others; one entry in 32 goes nowhere (a full expert)."""
    scores = _normal(g, 1, experts) + _normal(g, tokens, experts)
    chosen = scores.topk(k, dim=1).indices
    lost = torch.rand(tokens, k, generator=g, device="cuda") < 1.0 / 32
    return torch.where(lost, torch.full_like(chosen, experts), chosen).reshape(-1).contiguous()


def _order(chosen, experts):
    """offsets [experts + 1] and slots [entries]: where each entry goes when entries are ordered by expert, first come first."""
    held = chosen < experts
    key = torch.where(held, chosen, experts)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order).scatter_(0, order, torch.arange(order.numel(), device=order.device))
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=order.device).scatter_add_(0, key, torch.ones_like(key))
    ends = counts[:experts].cumsum(0)
    return torch.cat([ends.new_zeros(1), ends]), torch.where(held, place, _DROPPED)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["op"] == "topk":
        r, c, k = case["rows"], case["cols"], case["k"]
        if case["dir"] == "fwd":
            s["x"] = _normal(g, r, c, scale=3.0)
            s["values"], s["indices"] = _empty(r, k), _empty(r, k, dtype=torch.int64)
        else:
            perm, start = torch.randperm(c, generator=g, device="cuda"), torch.randint(c, (r, 1), generator=g, device="cuda")
            s["indices"] = perm[(start + torch.arange(k, device="cuda")) % c].contiguous()
            s["y_g"] = _normal(g, r, k, scale=1.0 / r)
            s["x_g"] = _normal(g, r, c, scale=1.0 / r) if case["acc"] else _empty(r, c)
            s["x_g0"] = s["x_g"].clone() if case["acc"] else None
    elif case["op"] == "distill":
        r, c, k = case["rows"], case["cols"], case["k"]
        x = _normal(g, r, c, scale=2.0)
        perm, start = torch.randperm(c, generator=g, device="cuda"), torch.randint(c, (r, 1), generator=g, device="cuda")
        s["indices"] = perm[(start + torch.arange(k, device="cuda")) % c].contiguous()
        s["teacher"] = _normal(g, r, k, scale=2.0).sort(dim=1, descending=True).values.add_(6.0).contiguous()
        x.scatter_add_(1, s["indices"], 0.5 * s["teacher"])  # a student that has learnt something
        s["logits"] = x
        s["w"] = None
        if case["weights"]:  # the mean over the real rows; one row in sixteen is padding
            real = torch.rand(r, generator=g, device="cuda") >= 1.0 / 16
            s["w"] = real.float() / real.sum().clamp(min=1)
        s["stats"], s["row_loss"], s["loss"] = _empty(r, 2), _empty(r), _empty(1)
        if case["dir"] == "bwd":
            s["stats"] = _stats(x, case["temp"])
        if case["dir"] != "fwd":
            s["grad"] = _normal(g, r, c, scale=1.0 / r) if case["acc"] else _empty(r, c)
            s["grad0"] = s["grad"].clone() if case["acc"] else None
    elif case["op"] == "experts":
        t, k, e, d = case["tokens"], case["k"], case["experts"], case["width"]
        n = t * k
        s["chosen"] = _choices(g, t, k, e)
        s["offsets"], s["slots"] = _empty(e + 1, dtype=torch.int64), _empty(n, dtype=torch.int64)
        if case["dir"] == "combine":
            s["offsets"], s["slots"] = _order(s["chosen"], e)
        if case["dir"] != "combine":
            s["x"], s["rows"] = _normal(g, t, d), _empty(n, d)
        if case["dir"] != "dispatch":
            s["y"], s["out"] = _normal(g, n, d), _empty(t, d)
            s["weights"] = torch.softmax(_normal(g, t, k), dim=1).contiguous()
        if case["dir"] == "train":
            s["out_g"], s["y_g"], s["weights_g"] = _normal(g, t, d, scale=1.0 / t), _empty(n, d), _empty(t, k)
            s["rows_g"], s["x_g"] = _normal(g, n, d, scale=1.0 / t), _empty(t, d)
    else:
        n, e, i, o = case["rows"], case["experts"], case["fan_in"], case["fan_out"]
        key = _choices(g, n, 1, e) if e > 1 else torch.zeros(n, dtype=torch.int64, device="cuda")
        offsets, _ = _order(key, e)
        s["offsets"], s["ends"] = offsets, offsets.tolist()
        s["x"], s["w"] = _normal(g, n, i), _normal(g, e, o, i, scale=math.sqrt(2.0 / i))
        s["b"] = _normal(g, e, o, scale=0.1) if case["bias"] else None
        if case["dir"] == "fwd":
            s["y"] = _empty(n, o)
        else:
            s["gy"], s["act_in"] = _normal(g, n, o, scale=1.0 / n), None
            if case["relu"]:
                s["x"] = s["act_in"] = s["x"].relu_()
            s["gw"], s["gb"], s["gx"] = _empty(e, o, i), (_empty(e, o) if case["bias"] else None), _empty(n, i)
    return s


def _stats(x, temp):
    top = x.amax(dim=1, keepdim=True)
    return torch.cat([top, ((x - top) / temp).exp().sum(dim=1, keepdim=True).log()], dim=1).contiguous()


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _OWN[s["op"]](s)
    return _PLAIN[s["op"]](s)


def _plain_topk(s):
    if s["dir"] == "fwd":
        # values that order like the floats in the upper half, later columns smaller in the lower: no two are the same
        bits = s["x"].view(torch.int32).to(torch.int64)
        key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 32) - torch.arange(s["cols"], device="cuda")
        at = key.topk(s["k"], dim=1).indices
        return {"values": s["x"].gather(1, at), "indices": at}
    if s["acc"]:
        return {"x_g": s["x_g0"].scatter_add(1, s["indices"], s["y_g"])}
    return {"x_g": torch.zeros_like(s["x_g"]).scatter_add_(1, s["indices"], s["y_g"])}


def _plain_distill(s):
    x, temp, at = s["logits"], s["temp"], s["indices"]
    w = s["w"] if s["w"] is not None else 1.0 / s["rows"]
    log_q = s["teacher"] / temp
    log_q = log_q - log_q.logsumexp(dim=1, keepdim=True)
    q = log_q.exp()
    stats = _stats(x, temp) if s["dir"] != "bwd" else s["stats"]
    out = {}
    if s["dir"] != "bwd":
        log_p = (x.gather(1, at) - stats[:, :1]) / temp - stats[:, 1:]
        row_loss = (q * (log_q - log_p)).sum(dim=1).mul_(temp * temp)
        if s["w"] is not None:
            row_loss = torch.where(s["w"] != 0, row_loss, 0.0)
        out.update(row_loss=row_loss, loss=(row_loss.double() * w).sum().float().reshape(1))
        if s["dir"] == "fwd":
            out["stats"] = stats if s["w"] is None else torch.where(s["w"].unsqueeze(1) != 0, stats, 0.0)
    if s["dir"] != "fwd":
        d = ((x - stats[:, :1]) / temp - stats[:, 1:]).exp_()
        d.scatter_add_(1, at, -q)
        d = d.mul_(w.unsqueeze(1) * temp) if s["w"] is not None else d.mul_(w * temp)
        out["grad"] = d.add_(s["grad0"]) if s["acc"] else d
    return out


def _plain_to_experts(s):
    t, k = s["tokens"], s["k"]
    offsets, slots = _order(s["chosen"], s["experts"])
    held = (slots >= 0).unsqueeze(1)
    rows = torch.zeros(t * k + 1, s["width"], device="cuda")  # the last row takes what goes nowhere
    rows[torch.where(slots >= 0, slots, t * k)] = s["x"].repeat_interleave(k, dim=0) * held
    return offsets, slots, rows[:-1]


def _plain_gather(rows, slots, tokens, k):
    got = rows[slots.clamp(min=0)] * (slots >= 0).unsqueeze(1)
    return got.reshape(tokens, k, -1)


def _plain_experts(s):
    t, k = s["tokens"], s["k"]
    out = {}
    slots = s["slots"]
    if s["dir"] != "combine":
        out["offsets"], out["slots"], out["rows"] = _plain_to_experts(s)
        slots = out["slots"]
    if s["dir"] != "dispatch":
        y = _plain_gather(s["y"], slots, t, k)
        out["out"] = (y * s["weights"].unsqueeze(2)).sum(dim=1)
    if s["dir"] == "train":
        out["weights_g"] = (y * s["out_g"].unsqueeze(1)).sum(dim=2)
        spread = (s["weights"].unsqueeze(2) * s["out_g"].unsqueeze(1)).reshape(t * k, -1)
        y_g = torch.zeros(t * k + 1, s["width"], device="cuda")
        y_g[torch.where(slots >= 0, slots, t * k)] = spread * (slots >= 0).unsqueeze(1)
        out["y_g"] = y_g[:-1]
        out["x_g"] = _plain_gather(s["rows_g"], slots, t, k).sum(dim=1)
    return out


def _plain_expert_linear(s):
    ends = s["ends"]
    if s["dir"] == "fwd":
        y = torch.zeros_like(s["y"])
        for e, (a, b) in enumerate(zip(ends, ends[1:])):
            if b > a:
                torch.mm(s["x"][a:b], s["w"][e].t(), out=y[a:b])
                if s["b"] is not None:
                    y[a:b] += s["b"][e]
        return {"y": y.relu_() if s["relu"] else y}
    gw, gx = torch.zeros_like(s["gw"]), torch.zeros_like(s["gx"])
    gb = torch.zeros_like(s["gb"]) if s["gb"] is not None else None
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if b > a:
            torch.mm(s["gy"][a:b].t(), s["x"][a:b], out=gw[e])
            torch.mm(s["gy"][a:b], s["w"][e], out=gx[a:b])
            if gb is not None:
                torch.sum(s["gy"][a:b], dim=0, out=gb[e])
    if s["act_in"] is not None:
        gx = torch.where(s["act_in"] > 0, gx, 0.0)
    return {"gw": gw, "gx": gx} if gb is None else {"gw": gw, "gb": gb, "gx": gx}


_PLAIN = {"topk": _plain_topk, "distill": _plain_distill, "experts": _plain_experts, "expert_linear": _plain_expert_linear}


# ---- the library's calls --------------------------------------------------------------------------------------
_DEVICE = []


def _device():
    if not _DEVICE:
        from zigrad_amd import HipDevice

        _DEVICE.append(HipDevice(torch.cuda.current_device()))
    return _DEVICE[0]


def _buffers(s):
    """The library's views of a state's tensors, made once: a program keeps its buffers in this form."""
    b = s.get("buffers")
    if b is None:
        from zigrad_amd import DevBuf

        kinds = {torch.float32: np.dtype(np.float32), torch.int64: np.dtype(np.uint64)}
        b = s["buffers"] = {n: DevBuf(v.data_ptr(), v.numel(), kinds[v.dtype], 0, "view") for n, v in s.items()
                            if isinstance(v, torch.Tensor)}
    return b


def _own_topk(s):
    dev, b = _device(), _buffers(s)
    size = {"rows": s["rows"], "cols": s["cols"], "k": s["k"]}
    if s["dir"] == "fwd":
        dev.dispatch("topk_fwd", x=b["x"], values=b["values"], indices=b["indices"], **size)
        return {"values": s["values"], "indices": s["indices"]}
    if s["acc"]:
        dev.mem_copy(b["x_g0"], b["x_g"])
    dev.dispatch("topk_bwd", indices=b["indices"], y_g=b["y_g"], x_g=b["x_g"], accumulate=s["acc"], **size)
    return {"x_g": s["x_g"]}


def _own_distill(s):
    dev, b = _device(), _buffers(s)
    p = {"logits": b["logits"], "teacher": b["teacher"], "indices": b["indices"], "weights": b.get("w"), "stats": b["stats"],
         "rows": s["rows"], "cols": s["cols"], "k": s["k"], "temperature": s["temp"]}
    if s["dir"] != "fwd" and s["acc"]:
        dev.mem_copy(b["grad0"], b["grad"])
    if s["dir"] == "fwd":
        dev.dispatch("distill_fwd", row_loss=b["row_loss"], loss=b["loss"], **p)
        return {"row_loss": s["row_loss"], "loss": s["loss"], "stats": s["stats"]}
    if s["dir"] == "bwd":
        dev.dispatch("distill_bwd", grad=b["grad"], accumulate=s["acc"], **p)
        return {"grad": s["grad"]}
    dev.dispatch("distill_fwd_bwd", row_loss=b["row_loss"], loss=b["loss"], grad=b["grad"], accumulate=s["acc"], **p)
    return {"row_loss": s["row_loss"], "loss": s["loss"], "grad": s["grad"]}


def _own_experts(s):
    dev, b = _device(), _buffers(s)
    size = {"n_tokens": s["tokens"], "k": s["k"], "width": s["width"]}
    out = {}
    if s["dir"] != "combine":
        dev.dispatch("expert_sort", experts=b["chosen"], offsets=b["offsets"], slots=b["slots"], n_experts=s["experts"])
        dev.dispatch("expert_dispatch", x=b["x"], slots=b["slots"], y=b["rows"], **size)
        out.update(offsets=s["offsets"], slots=s["slots"], rows=s["rows"])
    if s["dir"] != "dispatch":
        dev.dispatch("expert_combine", y=b["y"], slots=b["slots"], weights=b["weights"], out=b["out"], **size)
        out["out"] = s["out"]
    if s["dir"] == "train":
        dev.dispatch("expert_combine_bwd", out_g=b["out_g"], y=b["y"], slots=b["slots"], weights=b["weights"], y_g=b["y_g"],
                     weights_g=b["weights_g"], **size)
        dev.dispatch("expert_dispatch_bwd", y_g=b["rows_g"], slots=b["slots"], x_g=b["x_g"], accumulate=False, **size)
        out.update(y_g=s["y_g"], weights_g=s["weights_g"], x_g=s["x_g"])
    return out


def _own_expert_linear(s):
    dev, b = _device(), _buffers(s)
    size = {"n_rows": s["rows"], "n_experts": s["experts"], "fan_in": s["fan_in"], "fan_out": s["fan_out"]}
    if s["dir"] == "fwd":
        dev.dispatch("expert_linear_fwd", x=b["x"], w=b["w"], bias=b.get("b"), y=b["y"], offsets=b["offsets"], relu=s["relu"], **size)
        return {"y": s["y"]}
    dev.dispatch("expert_linear_bwd", gy=b["gy"], x=b["x"], w=b["w"], act_in=b.get("act_in"), gw=b["gw"], gb=b.get("gb"),
                 gx=b["gx"], offsets=b["offsets"], accumulate=False, **size)
    return {"gw": s["gw"], "gx": s["gx"]} if s["gb"] is None else {"gw": s["gw"], "gb": s["gb"], "gx": s["gx"]}


_OWN = {"topk": _own_topk, "distill": _own_distill, "experts": _own_experts, "expert_linear": _own_expert_linear}


# ---------------------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"topk": _exact_topk, "distill": _exact_distill, "experts": _exact_experts,
            "expert_linear": _exact_expert_linear}[case["op"]](s)


def _exact_topk(s):
    rows, k = s["rows"], s["k"]
    step = max(1, (1 << 26) // s["cols"])
    if s["dir"] == "fwd":
        got = [s["x"][r:r + step].double().sort(dim=1, descending=True, stable=True) for r in range(0, rows, step)]
        return {"values": torch.cat([v.values[:, :k] for v in got]), "indices": torch.cat([v.indices[:, :k] for v in got])}
    x_g = s["x_g0"].double() if s["acc"] else torch.zeros(rows, s["cols"], dtype=torch.float64, device="cuda")
    r = torch.arange(rows, device="cuda").unsqueeze(1).expand(rows, k)
    return {"x_g": x_g.index_put((r, s["indices"]), s["y_g"].double(), accumulate=True)}


def _exact_distill(s):
    step, parts = max(1, (1 << 27) // s["cols"]), []
    for r in range(0, s["rows"], step):
        of = slice(r, r + step)
        x, t, at = s["logits"][of].double(), s["teacher"][of].double(), s["indices"][of]
        w = s["w"][of].double() if s["w"] is not None else torch.full((x.shape[0],), 1.0 / s["rows"], dtype=torch.float64, device="cuda")
        temp = float(s["temp"])
        log_p, q = torch.log_softmax(x / temp, dim=1), torch.softmax(t / temp, dim=1)
        whole = torch.zeros_like(x).index_put((torch.arange(x.shape[0], device="cuda").unsqueeze(1).expand_as(at), at), q, accumulate=True)
        part = {}
        if s["dir"] != "bwd":
            kl = temp ** 2 * (q * (torch.log_softmax(t / temp, dim=1) - log_p.gather(1, at))).sum(dim=1)
            part["row_loss"] = torch.where(w != 0, kl, torch.zeros_like(kl))
            part["loss"] = (w * kl).sum().reshape(1)
        if s["dir"] == "fwd":
            top = x.max(dim=1).values
            part["stats"] = torch.stack([top, torch.logsumexp(x / temp, dim=1) - top / temp], dim=1) * (w != 0).unsqueeze(1)
        if s["dir"] != "fwd":
            part["grad"] = temp * w.unsqueeze(1) * (log_p.exp() - whole)
            if s["acc"]:
                part["grad"] += s["grad0"][of]
        parts.append(part)
    return {n: sum(p[n] for p in parts) if n == "loss" else torch.cat([p[n] for p in parts]) for n in parts[0]}


def _exact_experts(s):
    t, k, e, d = s["tokens"], s["k"], s["experts"], s["width"]
    chosen = s["chosen"].tolist()
    lists = [[] for _ in range(e)]
    for i, c in enumerate(chosen):
        if c < e:
            lists[c].append(i)
    offsets, slots = [0], [_DROPPED] * (t * k)
    for entries in lists:
        offsets.append(offsets[-1] + len(entries))
    for c, entries in enumerate(lists):
        for n, i in enumerate(entries):
            slots[i] = offsets[c] + n
    slots = torch.tensor(slots, device="cuda")
    entry = torch.nonzero(slots >= 0).squeeze(1)
    place, token = slots[entry], torch.div(entry, k, rounding_mode="floor")
    out = {}
    if s["dir"] != "combine":
        out = {"offsets": torch.tensor(offsets, device="cuda"), "slots": slots,
               "rows": torch.zeros(t * k, d, dtype=torch.float64, device="cuda").index_copy(0, place, s["x"].double()[token])}
    if s["dir"] != "dispatch":
        w = s["weights"].double().reshape(-1)[entry].unsqueeze(1)
        out["out"] = torch.zeros(t, d, dtype=torch.float64, device="cuda").index_add(0, token, w * s["y"].double()[place])
    if s["dir"] == "train":
        g = s["out_g"].double()[token]
        out["y_g"] = torch.zeros(t * k, d, dtype=torch.float64, device="cuda").index_copy(0, place, w * g)
        dots = (g * s["y"].double()[place]).sum(dim=1)
        out["weights_g"] = torch.zeros(t * k, dtype=torch.float64, device="cuda").index_copy(0, entry, dots).reshape(t, k)
        out["x_g"] = torch.zeros(t, d, dtype=torch.float64, device="cuda").index_add(0, token, s["rows_g"].double()[place])
    return out


def _exact_expert_linear(s):
    n, ends = s["rows"], s["ends"]
    owner = torch.full((n,), -1, dtype=torch.int64)
    for e in range(s["experts"]):
        owner[ends[e]:ends[e + 1]] = e
    owner = owner.cuda()
    if s["dir"] == "fwd":
        y = torch.zeros(n, s["fan_out"], dtype=torch.float64, device="cuda")
        for e in range(s["experts"]):
            at = torch.nonzero(owner == e).squeeze(1)
            v = s["x"][at].double() @ s["w"][e].double().t()
            v = v + s["b"][e].double() if s["b"] is not None else v
            y[at] = v.clamp(min=0) if s["relu"] else v
        return {"y": y}
    out = {"gw": torch.zeros(s["gw"].shape, dtype=torch.float64, device="cuda")}
    if s["gb"] is not None:
        out["gb"] = torch.zeros(s["gb"].shape, dtype=torch.float64, device="cuda")
    out["gx"] = torch.zeros(n, s["fan_in"], dtype=torch.float64, device="cuda")
    for e in range(s["experts"]):
        at = torch.nonzero(owner == e).squeeze(1)
        gy = s["gy"][at].double()
        out["gw"][e] = gy.t() @ s["x"][at].double()
        if s["gb"] is not None:
            out["gb"][e] = gy.sum(dim=0)
        out["gx"][at] = gy @ s["w"][e].double()
    if s["act_in"] is not None:
        out["gx"] *= s["act_in"] > 0
    return out
