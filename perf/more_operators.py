"""Attention between the qkv and the o projection as measurable cases.

* ``prepare`` -- RMSNorm of every query and key head, the position rotation,
  and the new keys and values into a paged 8-bit cache
  (``LoadedModule.prepare_qk``);
* ``prefill`` -- causal attention of whole prompts, packed one after another,
  with grouped heads (``LoadedModule.attention_prefill``);
* ``decode``  -- one query row of each sequence over the paged cache
  (``LoadedModule.attention_decode``);
* ``copy``    -- pages of every layer of a cache to other pages
  (``LoadedModule.copy_pages``).

The cache: pages of 64 tokens; of a page and a key/value head, 64 x D codes of
the keys and D x 64 (transposed) of the values, e4m3, with one power-of-two
scale each: the smallest 2^e, e >= -100, with 448 * 2^e at least the largest
magnitude.

``run`` computes them by elementary torch operations in 32 bits (``own``
false), or through the library (``own`` true); ``exact`` states the same
definitions in 64 bits.  The head layout 32 / 8 of 128 is the 6144 columns of
the benchmark's qkv projection, 4096 its context, 36 its layers; the others
are generic.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

CONTEXT, LAYERS = 4096, 36
PAGE = 64        # tokens of a page
EPS = 1e-6
TOP = 448.0      # e4m3's largest value


def listed():
    return [
        # One decode step of one sequence: pure latency.
        {"name": "prepare-1", "kind": "prepare", "m": 1, "seqs": 1, "past": 2000, "heads": 32, "kv": 8, "dim": 128,
         "dtype": "bf16", "packed": False, "cached": True},
        # An odd decode batch of sequences of all ages, rows in f32.
        {"name": "prepare-61", "kind": "prepare", "m": 61, "seqs": 61, "past": CONTEXT, "heads": 14, "kv": 2,
         "dim": 64, "dtype": "f32", "packed": False, "cached": True},
        # A full context of new prompts and continued ones.
        {"name": "prepare-4096", "kind": "prepare", "m": CONTEXT, "seqs": 5, "past": 700, "heads": 32, "kv": 8,
         "dim": 128, "dtype": "bf16", "packed": True, "cached": True},
        # A short question.
        {"name": "prefill-37", "kind": "prefill", "m": 37, "seqs": 1, "heads": 32, "kv": 8, "dim": 128},
        # Ragged prompts in one pass, narrow heads, seven queries' heads to a key's.
        {"name": "prefill-2001", "kind": "prefill", "m": 2001, "seqs": 9, "heads": 14, "kv": 2, "dim": 64},
        # One full context.
        {"name": "prefill-4096", "kind": "prefill", "m": CONTEXT, "seqs": 1, "heads": 32, "kv": 8, "dim": 128},
        # Prompts of about a context each, packed.
        {"name": "prefill-16384", "kind": "prefill", "m": 4 * CONTEXT, "seqs": 4, "heads": 32, "kv": 8, "dim": 128},
        # One sequence near the end of its context.
        {"name": "decode-1", "kind": "decode", "m": 1, "most": 4001, "heads": 32, "kv": 8, "dim": 128},
        # A serving batch of sequences of all lengths, one of them without a token.
        {"name": "decode-64", "kind": "decode", "m": 64, "most": CONTEXT, "heads": 32, "kv": 8, "dim": 128},
        # A few long documents, narrow heads.
        {"name": "decode-5", "kind": "decode", "m": 5, "most": 16 * CONTEXT, "heads": 14, "kv": 2, "dim": 64},
        # Copy on write of the last pages of a few forked sequences.
        {"name": "copy-6", "kind": "copy", "n": 6, "pages": 64, "layers": LAYERS, "kv": 8, "dim": 128},
        # Compacting: pages move down into the holes.
        {"name": "copy-200", "kind": "copy", "n": 200, "pages": 640, "layers": LAYERS, "kv": 8, "dim": 128},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _layout(rng):
    kv = rng.choice([1, 2, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8])
    return {"heads": heads, "kv": kv, "dim": rng.choice([64, 128, 128])}


def draw(rng):
    kind = rng.choice(["prepare", "prefill", "prefill", "decode", "decode", "copy"])
    lay = _layout(rng)
    if kind == "prepare":
        packed = rng.random() < 0.5
        m = _log(rng, 1, CONTEXT if packed else 256)
        return {"kind": kind, "m": m, "seqs": _log(rng, 1, min(m, 40)) if packed else m,
                "past": rng.choice([0, _log(rng, 1, CONTEXT)]) if packed else _log(rng, 1, CONTEXT), **lay,
                "dtype": rng.choice(["f32", "bf16"]), "packed": packed, "cached": rng.random() < 0.8}
    if kind == "prefill":
        seqs = _log(rng, 1, 24)
        return {"kind": kind, "m": max(seqs, _log(rng, 1, 2 * CONTEXT)), "seqs": seqs, **lay}
    if kind == "decode":
        most = _log(rng, 1, 16 * CONTEXT)
        size = 2 * lay["kv"] * lay["dim"] * most
        return {"kind": kind, "m": min(_log(rng, 1, 200), max(1, (CONTEXT * 64 * 2048) // size)), "most": most, **lay}
    n, layers = _log(rng, 1, 200), rng.choice([1, 4, LAYERS])
    return {"kind": kind, "n": n, "pages": 2 * n + _log(rng, 1, 200), "layers": layers, "kv": lay["kv"],
            "dim": lay["dim"]}


# ------------------------------------------------------------------ sizes: functions of the case alone
def _lengths(case):
    """Rows of each sequence of the batch."""
    if case["kind"] == "prepare" and not case["packed"]:
        return [1] * case["m"]
    rng = random.Random(case["m"] * 1000 + case["seqs"])
    cuts = sorted(rng.sample(range(1, case["m"]), case["seqs"] - 1)) if case["seqs"] > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [case["m"]])]


def _past(case):
    """Tokens that each sequence has in the cache already; packed, every other one is new."""
    rng = random.Random(case["past"] + 7 * case["m"])
    n = len(_lengths(case))
    if n == 1:
        return [case["past"]]
    return [0 if case["packed"] and i % 2 == 0 else rng.randint(0, case["past"]) for i in range(n)]


def _tokens(case):
    """Tokens that each decoded sequence sees."""
    rng = random.Random(case["most"] * 1000 + case["m"])
    n = [case["most"]] + [rng.randint(1, case["most"]) for _ in range(case["m"] - 1)]
    if case["m"] > 8:
        n[5] = 0
    return n


# ------------------------------------------------------------------ inputs
class _Inputs:
    def __init__(self, seed):
        self.gen = torch.Generator("cuda").manual_seed(seed)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.gen, device="cuda")

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def ints(self, v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    def table(self, counts, pages):
        """Pages of sequences that grew in turns: any order; -1 behind the last."""
        width = max(1, max(counts))
        order = torch.randperm(pages, generator=self.gen, device="cuda").int()
        at, rows = 0, []
        for c in counts:
            rows.append(torch.nn.functional.pad(order[at:at + c], (0, width - c), value=-1))
            at += c
        return torch.stack(rows)


def _held(x):
    """Blocks x[..., a, b] as the cache holds them: codes and scales."""
    s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((-2, -1)).clamp_min(1e-20).double() / TOP))).float()
    return (x / s[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8), s


def _cache(g, layers, pages, kv, dim):
    """A cache whose pages all hold tokens: keys with a few large channels."""
    codes = torch.empty(layers, pages, kv, 2, PAGE * dim, dtype=torch.uint8, device="cuda")
    scales = torch.empty(layers, pages, kv, 2, device="cuda")
    gain = 0.6 + 0.8 * g.uniform(kv, 1, dim)
    gain[:, :, ::29] *= 4.0
    for layer in range(layers):
        k, scales[layer, ..., 0] = _held(g.normal(pages, kv, PAGE, dim) * gain)
        v, scales[layer, ..., 1] = _held(g.normal(pages, kv, dim, PAGE))
        codes[layer, ..., 0, :], codes[layer, ..., 1, :] = k.flatten(2), v.flatten(2)
    return codes, scales


def _inputs(case, seed):
    """The case's inputs alone: a pure function of the case and the seed."""
    g, kv, dim = _Inputs(seed), case["kv"], case["dim"]
    if case["kind"] == "copy":
        codes, scales = _cache(g, case["layers"], case["pages"], kv, dim)
        at = torch.randperm(case["pages"], generator=g.gen, device="cuda").int()
        return {"codes": codes, "scales": scales, "src": at[:case["n"]].clone(),
                "dst": at[case["n"]:2 * case["n"]].clone()}
    m, heads = case["m"], case["heads"]
    if case["kind"] == "decode":
        tokens = _tokens(case)
        counts = [-(-t // PAGE) for t in tokens]
        pages = sum(counts) + 3
        codes, scales = _cache(g, 1, pages, kv, dim)
        return {"q": (1.5 * g.normal(m, heads, dim)).bfloat16(), "codes": codes, "scales": scales,
                "lengths": g.ints(tokens), "table": g.table(counts, pages)}
    rows = _lengths(case)
    starts = g.ints([0] + list(np.cumsum(rows)))
    if case["kind"] == "prefill":
        common = g.normal(1, kv, dim)  # what the queries share, and each prompt's first key answers to
        q = g.normal(m, heads, dim) + 0.5 * common.repeat_interleave(heads // kv, 1)
        k = g.normal(m, kv, dim)
        k[starts[:-1].long()] += common
        return {"q": (1.2 * q).bfloat16(), "k": k.bfloat16(), "v": g.normal(m, kv, dim).bfloat16(), "starts": starts,
                "rows": rows}
    past = _past(case)
    counts = [-(-(p + r) // PAGE) for p, r in zip(past, rows)]
    pages = sum(counts) + 3
    qkv = g.normal(m, (heads + 2 * kv) * dim)
    qkv[:, ::97] *= 6.0
    positions = max(p + r for p, r in zip(past, rows))
    angle = torch.arange(positions, device="cuda").double()[:, None] * \
        (1e6 ** (-torch.arange(dim // 2, device="cuda").double() * 2 / dim))
    i = {"qkv": qkv.bfloat16() if case["dtype"] == "bf16" else qkv.bfloat16().float(),
         "q_gain": 1.0 + 0.3 * g.normal(dim), "k_gain": 1.0 + 0.3 * g.normal(dim),
         "rope": torch.cat([angle.cos(), angle.sin()], 1).float(), "past": g.ints(past),
         "starts": starts if case["packed"] else None, "rows": rows, "pasts": past}
    if case["cached"]:
        codes, scales = _cache(g, 1, pages, kv, dim)
        i.update(codes=codes, scales=scales, table=g.table(counts, pages))
    return i


# ------------------------------------------------------------------ the plain forms
def _values(codes):
    return codes.view(torch.float8_e4m3fn).float()


def _as_e4m3(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _scale_for(most):
    """The smallest 2^e, e >= -100, with 448 * 2^e >= most."""
    part, e = torch.frexp(most)           # most = part * 2^e, part in [0.5, 1)
    e = torch.where(part > 0.875, e - 8, e - 9)
    return torch.ldexp(torch.ones_like(most), torch.where(most > 0, e, torch.full_like(e, -100)).clamp_min(-100))


def _plain_prepare(case, i, outs):
    m, heads, kv, dim = case["m"], case["heads"], case["kv"], case["dim"]
    row = torch.arange(m, device="cuda")
    if i["starts"] is None:
        seq, pos = row, i["past"].long()
    else:
        seq = torch.searchsorted(i["starts"][1:].contiguous(), row.int(), right=True)
        pos = i["past"][seq].long() + row - i["starts"][seq].long()
    x = i["qkv"].float().view(m, heads + 2 * kv, dim)
    v = x[:, heads + kv:]
    x = x[:, :heads + kv]
    gain = torch.cat([i["q_gain"].expand(heads, dim), i["k_gain"].expand(kv, dim)])
    x = x * torch.rsqrt((x * x).mean(2, keepdim=True) + EPS) * gain
    cos, sin = i["rope"][pos][:, None].chunk(2, 2)
    a, b = x.chunk(2, 2)
    x = torch.cat([a * cos - b * sin, b * cos + a * sin], 2)
    k = x[:, heads:]
    outs["q"].copy_(x[:, :heads])
    if "k" in outs:
        outs["k"].copy_(k)
        outs["v"].copy_(v)
    if not case["cached"]:
        return
    # the rows of one page: a run; runs of a batch in order
    slot = pos % PAGE
    first = torch.ones_like(row, dtype=torch.bool)
    first[1:] = (seq[1:] != seq[:-1]) | (slot[1:] == 0)
    run = first.cumsum(0) - 1
    runs = sum((p + r - 1) // PAGE - p // PAGE + 1 for p, r in zip(i["pasts"], i["rows"]))
    page = torch.zeros(runs, dtype=torch.long, device="cuda").index_copy_(
        0, run, i["table"][seq, pos // PAGE].long())
    old = torch.full((runs,), PAGE, device="cuda").scatter_reduce_(0, run, slot, "amin")
    new = torch.zeros(runs, PAGE, dtype=torch.bool, device="cuda").index_put_((run, slot), torch.ones((), dtype=torch.bool, device="cuda"))
    kept = torch.arange(PAGE, device="cuda") < old[:, None]
    codes, scales = i["codes"][0], i["scales"][0]
    for which, y in enumerate((k, v)):
        block = torch.zeros(runs, PAGE, kv, dim, device="cuda").index_put_((run, slot), y.contiguous())
        block = block.permute(0, 2, 1, 3)                                    # [runs, kv, PAGE, dim]
        was = torch.where((old > 0)[:, None], scales[page, :, which], torch.zeros_like(scales[page, :, which]))
        scale = torch.maximum(was, _scale_for(block.abs().amax((2, 3))))
        had = codes[page, :, which]
        had = had.view(runs, kv, PAGE, dim) if which == 0 else had.view(runs, kv, dim, PAGE).transpose(2, 3)
        again = _as_e4m3(_values(had.contiguous()) * (was / scale)[:, :, None, None])
        made = _as_e4m3(block / scale[:, :, None, None])
        made = torch.where(new[:, None, :, None], made, torch.where(kept[:, None, :, None], again, had))
        codes[page, :, which] = (made if which == 0 else made.transpose(2, 3)).reshape(runs, kv, -1)
        scales[page, :, which] = scale


def _plain_prefill(case, i, out):
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    at = 0
    for n in i["rows"]:
        q = i["q"][at:at + n].float().view(n, kv, -1, dim).permute(1, 2, 0, 3).reshape(kv, -1, dim)
        k = i["k"][at:at + n].float().permute(1, 2, 0).contiguous()
        v = i["v"][at:at + n].float().transpose(0, 1).contiguous()
        s = torch.matmul(q, k).view(kv, -1, n, n) * dim ** -0.5
        s = s.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu_(1), float("-inf"))
        s = torch.exp(s - s.amax(3, keepdim=True))
        s = (s / s.sum(3, keepdim=True)).view(kv, -1, n)
        out[at:at + n] = torch.matmul(s, v).view(kv, -1, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim)
        at += n


def _plain_decode(case, i, out):
    m, heads, kv, dim = case["m"], case["heads"], case["kv"], case["dim"]
    codes, scales = i["codes"][0], i["scales"][0]
    at = i["table"].long().clamp_min(0)
    width = at.shape[1]
    step = max(1, (1 << 28) // (width * PAGE * kv * dim))   # sequences at a time
    for b in range(0, m, step):
        t, n = at[b:b + step], len(at[b:b + step])
        k = _values(codes[t, :, 0]).view(n, width, kv, PAGE, dim) * scales[t, :, 0][..., None, None]
        v = _values(codes[t, :, 1]).view(n, width, kv, dim, PAGE) * scales[t, :, 1][..., None, None]
        k = k.permute(0, 2, 4, 1, 3).reshape(n, kv, dim, -1)
        v = v.permute(0, 2, 1, 4, 3).reshape(n, kv, -1, dim)
        s = torch.matmul(i["q"][b:b + step].float().view(n, kv, -1, dim), k) * dim ** -0.5
        dead = torch.arange(width * PAGE, device="cuda") >= i["lengths"][b:b + step, None, None, None]
        s = s.masked_fill_(dead, float("-inf"))
        s = torch.exp(s - s.amax(3, keepdim=True).nan_to_num(neginf=0.0))
        total = s.sum(3, keepdim=True)
        o = torch.matmul(s, v) / torch.where(total > 0, total, torch.ones_like(total))
        out[b:b + step] = o.reshape(n, heads, dim)


def _plain_copy(case, i):
    src, dst = i["src"].long(), i["dst"].long()
    i["codes"][:, dst] = i["codes"][:, src]
    i["scales"][:, dst] = i["scales"][:, src]


# ------------------------------------------------------------------ the library's calls
class Buffer:
    """A torch tensor as the device buffer that the operators take."""

    _NP = {torch.float32: np.float32, torch.bfloat16: np.uint16, torch.uint8: np.uint8, torch.int32: np.int32}

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


def _call(case, i, outs):
    """The call that a program makes, on buffers that it keeps."""
    from inferrous_amd import KvCache
    mod, stream = _runtime()
    b = {name: Buffer(t) for name, t in i.items() if isinstance(t, torch.Tensor)}
    o = {name: Buffer(t) for name, t in outs.items()}
    cache = None
    if "codes" in b:
        cache = KvCache.over(b["codes"], b["scales"], i["codes"].shape[0], i["codes"].shape[1], case["kv"], case["dim"])
    if case["kind"] == "copy":
        def call():
            mod.copy_pages(stream, cache, b["src"], b["dst"])
    elif case["kind"] == "decode":
        def call():
            mod.attention_decode(stream, b["q"], cache, b["lengths"], b["table"], case["heads"], o["out"])
    elif case["kind"] == "prefill":
        def call():
            mod.attention_prefill(stream, b["q"], b["k"], b["v"], case["heads"], case["kv"], case["dim"], o["out"],
                                  starts=b["starts"])
    else:
        def call():
            mod.prepare_qk(stream, b["qkv"], case["heads"], case["kv"], case["dim"], b["rope"], o["q"],
                           q_gain=b["q_gain"], k_gain=b["k_gain"], starts=b.get("starts"), past=b["past"],
                           k_out=o.get("k"), v_out=o.get("v"), cache=cache, table=b.get("table"), eps=EPS)
    return call


def _outputs(case, i):
    """The buffers that a program has the results in."""
    m, dim = case.get("m"), case["dim"]

    def empty(heads):
        return torch.zeros(m, heads, dim, dtype=torch.bfloat16, device="cuda")

    if case["kind"] == "copy":
        return {}
    if case["kind"] != "prepare":
        return {"out": empty(case["heads"])}
    outs = {"q": empty(case["heads"])}
    if case["packed"] or not case["cached"]:
        outs.update(k=empty(case["kv"]), v=empty(case["kv"]))
    return outs


def _answer(i, outs, changed):
    """Outputs, and the cache where the call writes it."""
    held = {"codes": i["codes"].view(torch.float8_e4m3fn), "scales": i["scales"]} if changed and "codes" in i else {}
    return {**outs, **held}


def prepare(case, seed):
    i = _inputs(case, seed)
    outs = _outputs(case, i)
    state = {"case": case, "inputs": i, "outs": outs, "answer": _answer(i, outs, case["kind"] in ("prepare", "copy"))}
    if own:
        state["call"] = _call(case, i, outs)
    return state


def run(state):
    if own:
        state["call"]()
        return state["answer"]
    case, i, outs = state["case"], state["inputs"], state["outs"]
    if case["kind"] == "prepare":
        _plain_prepare(case, i, outs)
    elif case["kind"] == "prefill":
        _plain_prefill(case, i, outs["out"])
    elif case["kind"] == "decode":
        _plain_decode(case, i, outs["out"])
    else:
        _plain_copy(case, i)
    return state["answer"]


# ------------------------------------------------------------------ the work
def work(case):
    kv, dim = case["kv"], case["dim"]
    if case["kind"] == "copy":
        return {"bytes": 2 * case["n"] * case["layers"] * kv * (2 * PAGE * dim + 8) + 8 * case["n"], "flops": 0}
    m, heads = case["m"], case["heads"]
    if case["kind"] == "decode":
        tokens = _tokens(case)
        pages = sum(-(-t // PAGE) for t in tokens)
        return {"bytes": 2 * sum(tokens) * kv * dim + pages * (8 * kv + 4) + m * (4 + 4 * heads * dim),
                "flops": 4 * sum(tokens) * heads * dim}
    rows = _lengths(case)
    if case["kind"] == "prefill":
        return {"bytes": 4 * m * (heads + kv) * dim + 4 * len(rows),
                "flops": 4 * heads * dim * sum(n * (n + 1) // 2 for n in rows)}
    size = 2 if case["dtype"] == "bf16" else 4
    kept = 2 * m * kv * dim if case["cached"] else 0
    both = 4 * m * kv * dim if case["packed"] or not case["cached"] else 0
    return {"bytes": m * (heads + 2 * kv) * dim * size + 2 * m * heads * dim + both + kept + 4 * m * dim,
            "flops": m * (heads + kv) * dim * 9 + 4 * m * kv * dim}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    i = _inputs(case, seed)
    if case["kind"] == "copy":
        codes, scales = i["codes"].cpu().numpy().copy(), i["scales"].cpu().numpy().copy()
        for s, d in zip(i["src"].tolist(), i["dst"].tolist()):
            codes[:, d], scales[:, d] = codes[:, s], scales[:, s]
        return {"codes": torch.from_numpy(codes).cuda().view(torch.float8_e4m3fn).double(),
                "scales": torch.from_numpy(scales).cuda().double()}
    return {"prepare": _exact_prepare, "prefill": _exact_prefill, "decode": _exact_decode}[case["kind"]](case, i)


def _exact_prefill(case, i):
    """Head by head, queries in blocks."""
    group, dim = case["heads"] // case["kv"], case["dim"]
    out = torch.zeros(case["m"], case["heads"], dim, dtype=torch.float64, device="cuda")
    bounds = i["starts"].tolist()
    for lo, hi in zip(bounds, bounds[1:]):
        for h in range(case["heads"]):
            k, v = (i[name][lo:hi, h // group].double() for name in ("k", "v"))
            kt = k.t().contiguous()
            for a in range(lo, hi, 2048):
                b = min(a + 2048, hi)
                logit = torch.mm(i["q"][a:b, h].double(), kt[:, :b - lo].contiguous()) / math.sqrt(dim)
                seen = torch.arange(lo, b, device="cuda")[None] <= torch.arange(a, b, device="cuda")[:, None]
                p = torch.softmax(torch.where(seen, logit, float("-inf")), 1)
                out[a:b, h] = torch.mm(p, v[:b - lo].contiguous())
    return {"out": out}


def _exact_decode(case, i):
    """Sequence by sequence."""
    group, kv, dim = case["heads"] // case["kv"], case["kv"], case["dim"]
    out = torch.zeros(case["m"], case["heads"], dim, dtype=torch.float64, device="cuda")
    for r, n in enumerate(i["lengths"].tolist()):
        if n == 0:
            continue
        at = i["table"][r, :-(-n // PAGE)].long()
        held = i["codes"][0, at].view(torch.float8_e4m3fn).double() * i["scales"][0, at].double()[..., None]
        for h in range(kv):
            k = held[:, h, 0].reshape(-1, dim)[:n]
            v = held[:, h, 1].reshape(len(at), dim, PAGE).transpose(1, 2).reshape(-1, dim)[:n].contiguous()
            q = i["q"][r, h * group:(h + 1) * group].double()
            p = torch.softmax(torch.mm(q, k.t().contiguous()) / math.sqrt(dim), 1)
            out[r, h * group:(h + 1) * group] = torch.mm(p, v)
    return {"out": out}


def _exact_prepare(case, i):
    """Sequence by sequence, and in each page by page."""
    heads, kv, dim, half = case["heads"], case["kv"], case["dim"], case["dim"] // 2
    rows = i["qkv"].double().reshape(case["m"], -1, dim)
    q = torch.empty(case["m"], heads, dim, dtype=torch.float64, device="cuda")
    k = torch.empty(case["m"], kv, dim, dtype=torch.float64, device="cuda")
    v = rows[:, heads + kv:]
    held = scales = None
    if case["cached"]:
        held, scales = i["codes"][0].view(torch.float8_e4m3fn).double(), i["scales"][0].double()
    at = 0
    for s, (n, p) in enumerate(zip(i["rows"], i["pasts"])):
        turn = i["rope"][p:p + n].double()
        z = torch.complex(turn[:, :half], turn[:, half:])[:, None]
        for out, lo, hi, gain in ((q, 0, heads, "q_gain"), (k, heads, heads + kv, "k_gain")):
            x = rows[at:at + n, lo:hi]
            x = x / torch.sqrt(torch.mean(x ** 2, 2, keepdim=True) + EPS) * i[gain].double()
            w = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * z
            out[at:at + n] = torch.cat([w.real, w.imag], 2)
        if held is not None:
            for page in range(p // PAGE, (p + n - 1) // PAGE + 1):
                lo, hi = max(p, page * PAGE), min(p + n, (page + 1) * PAGE)
                slot, take = lo - page * PAGE, slice(at + lo - p, at + hi - p)
                where = int(i["table"][s, page])
                for which, y in ((0, k[take]), (1, v[take])):
                    need = torch.exp2(torch.ceil(torch.log2(y.abs().amax((0, 2)).clamp_min(2.0 ** -200) / TOP)).clamp_min(-100))
                    was = scales[where, :, which] if slot else torch.zeros_like(need)
                    now = torch.maximum(need, was)
                    block = held[where, :, which]
                    block = block.view(kv, PAGE, dim) if which == 0 else block.view(kv, dim, PAGE).transpose(1, 2)
                    # (powers of two: these products are exact in 32 bits)
                    block[:, :slot] = (block[:, :slot] * (was / now)[:, None, None]).float().to(torch.float8_e4m3fn).double()
                    block[:, slot:slot + hi - lo] = (y / now[:, None]).float().to(torch.float8_e4m3fn).double().transpose(0, 1)
                    scales[where, :, which] = now
        at += n
    out = {"q": q}
    if case["packed"] or not case["cached"]:
        out.update(k=k, v=v.contiguous())
    if held is not None:
        out.update(codes=held[None], scales=scales[None])
    return out
