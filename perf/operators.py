"""Routed layers as measurable cases: the operators that give a row weights of
its own beside the shared W8A8 projections.

* ``route`` -- a router's logits to expert ids and weights
  (``LoadedModule.route_experts``): softmax or sigmoid scores, an optional
  balance bias that counts in the choice only, group-limited choice, top-k,
  renormalised weights;
* ``moe``   -- the routed experts' W8A8 SwiGLU products and their weighted sum
  (``LoadedModule.experts_mlp``);
* ``lora``  -- a W8A8 projection with a low-rank BF16 adapter per row beside
  it, many adapters in one call (``LoadedModule.linear_adapters``).

``run`` computes them by elementary torch operations in 32 bits (``own``
false), or through the library (``own`` true); ``exact`` states the same
definitions in 64 bits.  Widths are the ones of the benchmark and the tests
(hidden 4096, MLP 12288, 6144 = 4096 + 2 * 1024 columns of q, k and v, 5003 x
2000) or generic.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

HIDDEN, INTER, QKV, CONTEXT = 4096, 12288, 6144, 4096
GROUP = 128  # columns of an act row that share one quantization scale


def listed():
    return [
        # The router of one decode step of one sequence: pure latency.
        {"name": "route-1", "kind": "route", "m": 1, "experts": 128, "k": 8, "score": "softmax", "groups": 1,
         "top_groups": 1, "group_top": 1, "renorm": True, "scale": 1.0, "bias": False, "dtype": "bf16", "mask": False},
        # A decode batch with balance bias and group-limited choice.
        {"name": "route-64", "kind": "route", "m": 64, "experts": 256, "k": 8, "score": "sigmoid", "groups": 8,
         "top_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5, "bias": True, "dtype": "f32", "mask": False},
        # Odd counts everywhere; experts that are switched off, and rows that none is left for.
        {"name": "route-999", "kind": "route", "m": 999, "experts": 60, "k": 6, "score": "softmax", "groups": 6,
         "top_groups": 3, "group_top": 1, "renorm": False, "scale": 1.0, "bias": False, "dtype": "f32", "mask": True},
        # Four full contexts of prompts in one pass.
        {"name": "route-16384", "kind": "route", "m": 4 * CONTEXT, "experts": 256, "k": 8, "score": "sigmoid",
         "groups": 8, "top_groups": 4, "group_top": 2, "renorm": True, "scale": 2.5, "bias": True, "dtype": "f32",
         "mask": False},
        # One sequence's decode step: eight experts' weights stream once.
        {"name": "moe-1", "kind": "moe", "m": 1, "hidden": HIDDEN, "inter": 1024, "experts": 64, "k": 8,
         "drop": False, "residual": False},
        # A decode batch: most experts are met, by one or two rows each.
        {"name": "moe-16", "kind": "moe", "m": 16, "hidden": 2048, "inter": 768, "experts": 128, "k": 8,
         "drop": False, "residual": False},
        # A short prompt, ragged in every dimension, slots without an expert, into the residual stream.
        {"name": "moe-333", "kind": "moe", "m": 333, "hidden": 2000, "inter": 720, "experts": 20, "k": 3,
         "drop": True, "residual": True},
        # A full context of prompts.
        {"name": "moe-4096", "kind": "moe", "m": CONTEXT, "hidden": HIDDEN, "inter": 1024, "experts": 64, "k": 8,
         "drop": False, "residual": False},
        # One request with an adapter on a square projection.
        {"name": "lora-1", "kind": "lora", "m": 1, "n": HIDDEN, "k": HIDDEN, "rank": 16, "adapters": 4,
         "runs": False, "residual": False},
        # A decode batch of requests with forty adapters, some with none, on q, k and v.
        {"name": "lora-64", "kind": "lora", "m": 64, "n": QKV, "k": HIDDEN, "rank": 32, "adapters": 40,
         "runs": False, "residual": False},
        # Ragged in every dimension, into the residual stream.
        {"name": "lora-77", "kind": "lora", "m": 77, "n": 5003, "k": 2000, "rank": 24, "adapters": 9,
         "runs": True, "residual": True},
        # A full context of a few requests' prompts through the down projection.
        {"name": "lora-4096", "kind": "lora", "m": CONTEXT, "n": HIDDEN, "k": INTER, "rank": 64, "adapters": 6,
         "runs": True, "residual": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


_MOST = 6 * CONTEXT * 8 * HIDDEN * 1024  # operations of moe-4096, the largest listed case
_MOST_BYTES = 64 * 3 * HIDDEN * 1024
_NEVER = (1536, 3072)


def draw(rng):
    while True:
        case = _draw(rng)
        if not any(v in _NEVER for v in case.values() if type(v) is int):
            return case


def _draw(rng):
    kind = rng.choice(["route", "moe", "moe", "lora", "lora"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 6, 8])
        experts = groups * max(2, _log(rng, 8, 384) // groups)
        top_groups = rng.randint(1, groups)
        k = min(rng.randint(1, 12), top_groups * (experts // groups))
        sigmoid = rng.random() < 0.5
        return {"kind": kind, "m": _log(rng, 1, 4 * CONTEXT), "experts": experts, "k": k,
                "score": "sigmoid" if sigmoid else "softmax", "groups": groups, "top_groups": top_groups,
                "group_top": rng.choice([1, 2]), "renorm": rng.random() < 0.7,
                "scale": rng.choice([1.0, 1.0, 2.5]), "bias": rng.random() < (0.8 if sigmoid else 0.3),
                "dtype": rng.choice(["f32", "bf16"]), "mask": rng.random() < 0.3}
    if kind == "moe":
        while True:
            m, experts = _log(rng, 1, CONTEXT), _log(rng, 2, 160)
            hidden, inter = 16 * _log(rng, 16, 256), 16 * _log(rng, 8, 128)
            if rng.random() < 0.5:
                hidden, inter = -(-hidden // 256) * 256, -(-inter // 128) * 128
            k = rng.randint(1, min(8, experts))
            if 6 * m * k * hidden * inter <= _MOST and 3 * experts * hidden * inter <= _MOST_BYTES:
                break
        return {"kind": kind, "m": m, "hidden": hidden, "inter": inter, "experts": experts, "k": k,
                "drop": rng.random() < 0.3, "residual": rng.random() < 0.4}
    while True:
        m, n, k = _log(rng, 1, CONTEXT), _log(rng, 64, 2 * INTER), 16 * _log(rng, 16, INTER // 16)
        if rng.random() < 0.5:
            k = -(-k // 128) * 128
        if 2 * m * n * k <= _MOST // 2:
            break
    return {"kind": kind, "m": m, "n": n, "k": k, "rank": rng.choice([8, 16, 16, 24, 32, 64, 128]),
            "adapters": _log(rng, 1, 96), "runs": rng.random() < 0.5, "residual": rng.random() < 0.4}


# ------------------------------------------------------------------ inputs
_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


class _Inputs:
    def __init__(self, seed):
        self.gen = torch.Generator("cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def rows(self, m, k):
        """BF16-valued activations with a few large channels."""
        x = self.normal(m, k)
        x[:, torch.randint(0, k, (max(1, k // 512),), generator=self.gen, device="cuda")] *= 8.0
        return x.bfloat16()

    def matrix(self, *shape, size=1.0):
        """int8 weights [..., n, k] of about 3.5 deviations per row, and the
        scales that make a row's products about ``size``."""
        w = torch.empty(shape, dtype=torch.int8, device="cuda")
        for part in w.view(-1, shape[-2], shape[-1]):
            part.copy_(self.normal(*part.shape).mul_(36.0).round_().clamp_(-127.0, 127.0))
        return w, (0.8 + 0.4 * self.uniform(*shape[:-1])) * (size / (36.0 * shape[-1] ** 0.5))


def _codes(x):
    """The framework's activation quantization of BF16 rows."""
    x = x.float()
    s = x.abs().amax(1).clamp_min(1e-8) / 127.0
    return (x / s[:, None]).round().clamp_(-127.0, 127.0).to(torch.int8), s


def _route_inputs(case, g):
    """Logits of a router: some experts more popular than others.  Rows whose
    choice 32 bits cannot tell apart (two of the best scores, or the last group
    in and the first out, within 4e-6 of their size but not equal) have no one
    right answer and are drawn again."""
    m, e = case["m"], case["experts"]
    popular = 0.5 * g.normal(e)
    bias = (0.001 * (100.0 * g.normal(e)).round()) if case["bias"] else None  # steps of a balance update

    def fresh(rows):
        x = 1.5 * g.normal(rows, e) + popular
        if case["mask"]:
            x[:, ::7] = float("-inf")                         # switched off for every row
            x.masked_fill_(g.uniform(rows, 1) < 0.02, float("-inf"))  # rows that no expert is left for
        return x.to(_DTYPE[case["dtype"]])

    logits = fresh(m)
    while True:
        near = _near(case, logits.double(), None if bias is None else bias.double())
        at = near.nonzero()[:, 0]
        if at.numel() == 0:
            return logits, bias
        logits[at] = fresh(at.numel())


def _near(case, x, bias):
    s, c = _scores(case, x, bias)
    c, grouped = _in_groups(case, c)

    def close(v, n):
        """Of the n + 1 best, any two neighbours (or for a set: only the last) near."""
        v = v.sort(1, descending=True).values[:, :n + 1]
        gap, size = v[:, :-1] - v[:, 1:], v.abs().nan_to_num(posinf=0.0, neginf=0.0)
        return (gap > 0) & (gap < 4e-6 * torch.maximum(size[:, :-1], size[:, 1:]) + 1e-30)

    near = close(c, case["k"]).any(1)
    if grouped is not None and case["top_groups"] < case["groups"]:
        near |= close(grouped, case["top_groups"])[:, -1]
    return near


def _inputs(case, seed):
    """The case's inputs alone: a pure function of the case and the seed."""
    g, m = _Inputs(seed), case["m"]
    if case["kind"] == "route":
        logits, bias = _route_inputs(case, g)
        return {"logits": logits, "bias": bias}
    if case["kind"] == "moe":
        e, h, f, k = case["experts"], case["hidden"], case["inter"], case["k"]
        q, asc = _codes(g.rows(m, h))
        s = torch.softmax(1.5 * g.normal(m, e) + 0.5 * g.normal(e), 1)
        top = s.topk(k, 1)
        weights, ids = top.values / top.values.sum(1, keepdim=True), top.indices.int()
        if case["drop"]:
            off = g.uniform(m, k) < 0.1
            off |= g.uniform(m, 1) < 0.02
            ids, weights = ids.masked_fill(off, -1), weights.masked_fill(off, 0.0)
        gate, up, down = g.matrix(e, f, h), g.matrix(e, f, h), g.matrix(e, h, f, size=0.5)
        return {"q": q, "asc": asc, "ids": ids, "weights": weights, "gate": gate, "up": up, "down": down,
                "residual": g.rows(m, h).float() if case["residual"] else None}
    n, k, r, a = case["n"], case["k"], case["rank"], case["adapters"]
    x = g.rows(m, k)
    q, asc = _codes(x)
    ids = torch.randint(-1, a, (m,), generator=g.gen, device="cuda", dtype=torch.int32)  # -1: the shared weights alone
    if case["runs"]:  # requests of several rows each
        ids = ids[torch.randint(0, m, (m,), generator=g.gen, device="cuda").div(max(1, m // 8), rounding_mode="floor")
                  .sort().values]
    return {"x": x, "q": q, "asc": asc, "w": g.matrix(n, k), "ids": ids,
            "a": (g.normal(a, r, k) * k ** -0.5).bfloat16(), "b": (0.05 * g.normal(a, n, r)).bfloat16(),
            "scaling": 2.0 * (0.5 + g.uniform(a)),
            "residual": g.rows(m, n).float() if case["residual"] else None}


# ------------------------------------------------------------------ the plain forms
def _scores(case, x, bias):
    """Scores s and choice scores c; an expert whose logit is -inf or NaN is out
    (c = -inf)."""
    x = x.nan_to_num(nan=float("-inf"), posinf=float("inf"), neginf=float("-inf"))
    out = x == float("-inf")
    if case["score"] == "softmax":
        top = x.amax(1, keepdim=True).nan_to_num(neginf=0.0)
        s = torch.exp(x - top)
        s = s / s.sum(1, keepdim=True).clamp_min(1e-30)
    else:
        s = 1.0 / (1.0 + torch.exp(-x))
    c = s if bias is None else s + bias
    return s, c.masked_fill(out, float("-inf"))


def _in_groups(case, c):
    """c with the experts outside the best groups out, and the groups' scores: the
    largest choice score of a group, or the sum of its two largest."""
    if case["groups"] == 1:
        return c, None
    parts = c.view(c.shape[0], case["groups"], -1)
    best = parts.sort(2, descending=True).values[:, :, :case["group_top"]]
    live = best[:, :, 0] > float("-inf")
    grouped = best.nan_to_num(neginf=0.0).sum(2).masked_fill(~live, float("-inf"))
    keep = grouped.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
    kept = torch.zeros_like(grouped, dtype=torch.bool).scatter_(1, keep, True)
    return parts.masked_fill(~kept[:, :, None], float("-inf")).reshape(c.shape), grouped


def _plain_route(case, i):
    s, c = _scores(case, i["logits"].float(), i["bias"])
    c = _in_groups(case, c)[0]
    c, ids = c.sort(dim=1, descending=True, stable=True)
    c, ids = c[:, :case["k"]], ids[:, :case["k"]]
    gone = c == float("-inf")
    w = s.gather(1, ids).masked_fill(gone, 0.0)
    if case["renorm"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
    return [ids.masked_fill(gone, -1).int(), w * case["scale"]]


def _act_codes(act):
    """Codes and scales of act rows, one scale to GROUP columns."""
    rows, f = act.shape
    parts = torch.nn.functional.pad(act, (0, -f % GROUP)).view(rows, -1, GROUP)
    s = parts.abs().amax(2, keepdim=True).clamp_min(1e-8) / 127.0
    return (parts / s).round().clamp_(-127.0, 127.0), s


def _expert(q, asc, wg, sg, wu, su, wd, sd):
    """One expert's SwiGLU MLP over its rows."""
    gate, up = (q @ wg.t()) * asc * sg, (q @ wu.t()) * asc * su
    codes, s = _act_codes(gate / (1.0 + torch.exp(-gate)) * up)
    return ((codes * s).flatten(1)[:, :wd.shape[1]] @ wd.t()) * sd


def _plain_moe(case, i, dt=torch.float32):
    m, k = i["ids"].shape
    out = torch.zeros(m, case["hidden"], dtype=dt, device="cuda")
    ids, weights, q, asc = i["ids"], i["weights"].to(dt), i["q"].to(dt), i["asc"].to(dt)[:, None]
    mats = (*i["gate"], *i["up"], *i["down"])
    for e in range(case["experts"]) if m * k > 16 else ids.flatten().unique().tolist():
        row, slot = (ids == e).nonzero(as_tuple=True)
        if e < 0 or row.numel() == 0:
            continue
        y = _expert(q[row], asc[row], *(t[e].to(dt) for t in mats))
        out.index_add_(0, row, y * weights[row, slot][:, None])  # a row meets an expert once
    return out if i["residual"] is None else out + i["residual"]


def _plain_lora(case, i):
    y = (i["q"].float() @ i["w"][0].float().t()) * i["asc"][:, None] * i["w"][1]
    if case["m"] <= 64:  # every row's own matrices
        at = i["ids"].clamp_min(0).long()
        h = (i["a"][at].float() * i["x"].float()[:, None, :]).sum(2)
        d = (i["b"][at].float() * h[:, None, :]).sum(2) * i["scaling"][at][:, None]
        y += torch.where((i["ids"] >= 0)[:, None], d, torch.zeros_like(d))
    else:
        for a in range(case["adapters"]):
            row = (i["ids"] == a).nonzero()[:, 0]
            if row.numel():
                y[row] += (i["x"][row].float() @ i["a"][a].float().t()) @ i["b"][a].float().t() * i["scaling"][a]
    return y if i["residual"] is None else y + i["residual"]


# ------------------------------------------------------------------ the library's calls
class Buffer:
    """A torch tensor as the device buffer that the operators take."""

    _NP = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.int8: np.int8, torch.int32: np.int32}

    def __init__(self, tensor):
        self.tensor = tensor
        self.dtype = np.dtype(self._NP[tensor.dtype])
        self.n = tensor.numel()
        self.nbytes = self.n * self.dtype.itemsize
        self.ptr = tensor.data_ptr()

    def __len__(self):
        return self.n


_RUNTIME = []


def _runtime():
    if not _RUNTIME:
        from inferrous_amd import CudaContext, load
        ctx = CudaContext.new(0)
        _RUNTIME.extend((load(ctx), ctx.default_stream()))
    return _RUNTIME


def _call(case, i):
    """The call that a program makes, on buffers that it keeps."""
    mod, stream = _runtime()
    b = {}
    for name, t in i.items():
        b[name] = tuple(map(Buffer, t)) if isinstance(t, tuple) else None if t is None else Buffer(t)
    m = case["m"]
    if case["kind"] == "route":
        ids = torch.empty(m, case["k"], dtype=torch.int32, device="cuda")
        weights = torch.empty(m, case["k"], device="cuda")
        outs = [Buffer(ids), Buffer(weights)]

        def call():
            mod.route_experts(stream, b["logits"], case["experts"], *outs, score=case["score"], bias=b["bias"],
                              groups=case["groups"], top_groups=case["top_groups"], group_top=case["group_top"],
                              renorm=case["renorm"], scale=case["scale"])
    elif case["kind"] == "moe":
        outs = [Buffer(torch.empty(m, case["hidden"], dtype=torch.bfloat16, device="cuda"))]

        def call():
            mod.experts_mlp(stream, b["q"], b["asc"], case["hidden"], b["ids"], b["weights"], *b["gate"], *b["up"],
                            *b["down"], case["experts"], outs[0], residual=b["residual"])
    else:
        outs = [Buffer(torch.empty(m, case["n"], dtype=torch.bfloat16, device="cuda"))]

        def call():
            mod.linear_adapters(stream, b["q"], b["asc"], *b["w"], case["k"], b["x"], b["ids"], b["a"], b["b"],
                                b["scaling"], outs[0], residual=b["residual"])
    return call, [o.tensor for o in outs]


def prepare(case, seed):
    state = {"case": case, "inputs": _inputs(case, seed)}
    if own:
        state["call"], state["outs"] = _call(case, state["inputs"])
    return state


def run(state):
    if own:
        state["call"]()
        return state["outs"]
    case, i = state["case"], state["inputs"]
    if case["kind"] == "route":
        return _plain_route(case, i)
    y = _plain_moe(case, i) if case["kind"] == "moe" else _plain_lora(case, i)
    return [y.bfloat16()]


# ------------------------------------------------------------------ the work
def work(case):
    m = case["m"]
    if case["kind"] == "route":
        e, k = case["experts"], case["k"]
        return {"bytes": m * (e * (4 if case["dtype"] == "f32" else 2) + 8 * k) + (4 * e if case["bias"] else 0),
                "flops": m * e * (4 + k)}
    if case["kind"] == "moe":
        h, f, e, k = case["hidden"], case["inter"], case["experts"], case["k"]
        met = e * (1.0 - (1.0 - k / e) ** m)  # experts that some row meets
        return {"bytes": int(met * (3 * h * f + 8 * f + 4 * h)) + m * (3 * h + 4 + 8 * k
                                                                       + (4 * h if case["residual"] else 0)),
                "flops": 6 * m * k * h * f}
    n, k, r, a = case["n"], case["k"], case["rank"], case["adapters"]
    met = a * (1.0 - (1.0 - 1.0 / (a + 1)) ** (min(m, 8) if case["runs"] else m))
    return {"bytes": n * k + 4 * n + int(met * 2 * r * (n + k)) + m * (3 * k + 8 + 2 * n
                                                                      + (4 * n if case["residual"] else 0)),
            "flops": 2 * m * (n * k + r * (n + k))}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    i = _inputs(case, seed)
    if case["kind"] == "route":
        return _exact_route(case, i)
    y = _exact_moe(case, i) if case["kind"] == "moe" else _exact_lora(case, i)
    return [y]


def _exact_route(case, i):
    x = i["logits"].double().cpu().numpy()
    m, e = x.shape
    k, per = case["k"], e // case["groups"]
    x = np.where(np.isnan(x), -np.inf, x)
    live = x > -np.inf
    if case["score"] == "softmax":
        top = np.where(live.any(1), x.max(1), 0.0)[:, None]
        s = np.exp(x - top)
        s = s / np.maximum(s.sum(1, keepdims=True), np.finfo(np.float64).tiny)
    else:
        s = 1.0 / (1.0 + np.exp(-x))
    c = np.where(live, s + (0.0 if i["bias"] is None else i["bias"].double().cpu().numpy()), -np.inf)
    if case["groups"] > 1:
        order = -np.sort(-c.reshape(m, -1, per), axis=2)
        score = order[:, :, 0].copy()
        if case["group_top"] == 2 and per > 1:
            score += np.where(order[:, :, 1] > -np.inf, order[:, :, 1], 0.0)
        rank = np.argsort(np.argsort(-score, axis=1, kind="stable"), axis=1, kind="stable")
        c = np.where(np.repeat(rank < case["top_groups"], per, axis=1), c, -np.inf)
    ids = np.argsort(-c, axis=1, kind="stable")[:, :k]
    gone = ~(np.take_along_axis(c, ids, 1) > -np.inf)
    w = np.where(gone, 0.0, np.take_along_axis(s, ids, 1))
    if case["renorm"]:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return [torch.from_numpy(np.where(gone, -1, ids).astype(np.int32)).cuda(), torch.from_numpy(w * case["scale"]).cuda()]


def _exact_moe(case, i):
    """Slot by slot: each row's slot s through its expert, experts in turn."""
    m, f = case["m"], case["inter"]
    total = torch.zeros(m, case["hidden"], dtype=torch.float64, device="cuda")
    if i["residual"] is not None:
        total += i["residual"].double()
    x = i["q"].double() * i["asc"].double()[:, None]
    for e in range(case["experts"]):
        coeff = (i["weights"].double() * (i["ids"] == e)).sum(1)
        at = torch.where((i["ids"] == e).any(1))[0]
        if len(at) == 0:
            continue
        gate = torch.mm(x[at], (i["gate"][0][e].double() * i["gate"][1][e].double()[:, None]).t().contiguous())
        up = torch.mm(x[at], (i["up"][0][e].double() * i["up"][1][e].double()[:, None]).t().contiguous())
        act = up * gate * torch.sigmoid(gate)
        held = torch.empty_like(act)
        for c in range(0, f, GROUP):
            part = act[:, c:c + GROUP]
            step = part.abs().max(1, keepdim=True).values.clamp(min=1e-8) / 127
            held[:, c:c + GROUP] = torch.round(part / step).clamp(-127, 127) * step
        y = torch.mm(held, (i["down"][0][e].double() * i["down"][1][e].double()[:, None]).t().contiguous())
        total[at] += coeff[at, None] * y
    return total


def _exact_lora(case, i):
    w = i["w"][0].double() * i["w"][1].double()[:, None]
    total = torch.mm(i["q"].double() * i["asc"].double()[:, None], w.t().contiguous())
    if i["residual"] is not None:
        total += i["residual"].double()
    for a in i["ids"].unique().tolist():
        if a >= 0:
            mine = (i["ids"] == a)[:, None]
            low = torch.mm(i["x"].double() * mine, i["a"][a].double().t().contiguous())
            total += torch.mm(low, i["b"][a].double().t().contiguous()) * i["scaling"][a].double()
    return total
