"""Cases and plain forms of the operators on local shards: embedding lookup and its gradient, conversion of rows to 8 bits,
the 8-bit product, and the products grouped by expert.

Where ``own`` is false ``run`` computes the plain form with elementary torch operations in 32 bits; where it is true it
makes the calls that a user of etha_amd makes.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
DEVICE = "cuda"


def listed():
    return [
        # a decoding step of one sequence: one row out of one TP rank's half of a 128256-row embedding
        {"name": "lookup 1 token", "op": "lookup", "tokens": 1, "vocab": 128256, "rows": 64128, "first": 0, "width": 4096,
         "dtype": "bf16", "out": "bf16", "ids": "i64", "scale": 1.0},
        # a prefill batch on the uneven tail shard of a 151936-row embedding over 6 ranks, fp32 masters read as bf16, scaled by
        # the square root of the width; five of six tokens are other ranks' and give zero rows
        {"name": "lookup prefill, tail shard", "op": "lookup", "tokens": 16381, "vocab": 151936, "rows": 25321, "first": 126615,
         "width": 4096, "dtype": "f32", "out": "bf16", "ids": "i32", "scale": 64.0},
        # a short micro-batch's gradient of a narrow vocabulary shard with a width that is no multiple of a vector
        {"name": "lookup gradient, short", "op": "lookup_grad", "tokens": 509, "vocab": 32000, "rows": 4000, "first": 8000,
         "width": 1001, "dtype": "bf16", "out": "f32", "ids": "i64", "scale": 1.0},
        # a training step's gradient of the whole 128256-row embedding
        {"name": "lookup gradient, large", "op": "lookup_grad", "tokens": 65536, "vocab": 128256, "rows": 128256, "first": 0,
         "width": 4096, "dtype": "bf16", "out": "bf16", "ids": "i64", "scale": 1.0},
        # the smallest projection of a decoder layer after a weight transfer (kv projection, one TP rank of two)
        {"name": "8-bit rows, kv projection", "op": "quantize", "rows": 512, "width": 4096, "dtype": "bf16"},
        # the largest one: an output head's shard in fp32
        {"name": "8-bit rows, output head", "op": "quantize", "rows": 64128, "width": 4096, "dtype": "f32"},
        # one token through an 8-bit up projection
        {"name": "8-bit product 1 token", "op": "int8", "tokens": 1, "out_width": 14336, "width": 4096, "dtype": "bf16", "bias": False},
        # a prefill batch through it, an odd number of tokens
        {"name": "8-bit product prefill", "op": "int8", "tokens": 8191, "out_width": 14336, "width": 4096, "dtype": "bf16", "bias": True},
        # a decoding step of eight sequences, two experts each: one TP rank of four of the experts' first matrix
        {"name": "experts decode", "op": "grouped", "tokens": 16, "experts": 8, "out_width": 3584, "width": 4096, "dtype": "bf16",
         "skew": 1.0},
        # a prefill batch over the same shard, uneven experts
        {"name": "experts prefill", "op": "grouped", "tokens": 16384, "experts": 8, "out_width": 3584, "width": 4096, "dtype": "bf16",
         "skew": 1.5},
        # both gradients of a small expert set with odd sizes, fp32 weight gradients
        {"name": "experts gradients, odd", "op": "grouped_grad", "tokens": 301, "experts": 8, "out_width": 515, "width": 258,
         "dtype": "f16", "out": "f32", "skew": 1.0},
        # both gradients of a training step
        {"name": "experts gradients, large", "op": "grouped_grad", "tokens": 16384, "experts": 8, "out_width": 3584, "width": 4096,
         "dtype": "bf16", "out": "bf16", "skew": 1.0},
    ]


def _log_int(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; half of them as they fall, half rounded to a multiple of 64 where that is possible."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    return v // 64 * 64 if v >= 128 and v // 64 * 64 >= lo and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "quantize", "int8", "grouped", "grouped_grad"])
    if op in ("lookup", "lookup_grad"):
        vocab = _log_int(rng, 1000, 128256)
        rows = max(1, vocab // rng.choice([1, 1, 2, 4, 6, 8]))
        case = {"op": op, "tokens": _log_int(rng, 1, 65536), "vocab": vocab, "rows": rows, "first": rng.choice([0, vocab - rows]),
                "width": _log_int(rng, 64, 4096), "dtype": rng.choice(["bf16", "bf16", "f32", "f16"]), "ids": rng.choice(["i32", "i64"]),
                "scale": rng.choice([1.0, 64.0, 0.125])}
        same = case["dtype"]
        case["out"] = rng.choice(["f32", same]) if op == "lookup_grad" else rng.choice(["bf16", same])
        if case["out"] == "f32" and op == "lookup_grad":
            case["rows"] = min(rows, 64128)
            case["first"] = min(case["first"], vocab - case["rows"])
        if case["dtype"] == "f32":
            case["tokens"] = min(case["tokens"], 32768)
        return case
    if op == "quantize":
        return {"op": op, "rows": _log_int(rng, 1, 64128), "width": _log_int(rng, 64, 4096), "dtype": rng.choice(["bf16", "f32", "f16"])}
    if op == "int8":
        return {"op": op, "tokens": _log_int(rng, 1, 8191), "out_width": _log_int(rng, 64, 14336), "width": _log_int(rng, 64, 4096),
                "dtype": rng.choice(["bf16", "f16", "f32"]), "bias": rng.random() < 0.5}
    case = {"op": op, "tokens": _log_int(rng, 1, 16384), "experts": rng.choice([1, 3, 8, 8, 16, 64]), "out_width": _log_int(rng, 64, 3584),
            "width": _log_int(rng, 64, 4096), "dtype": rng.choice(["bf16", "f16"]), "skew": rng.choice([0.0, 1.0, 2.0])}
    if case["experts"] > 8:  # many experts are narrow ones
        case["out_width"], case["width"] = min(case["out_width"], 1536), min(case["width"], 2048)
    if op == "grouped_grad":
        case["out"] = rng.choice(["f32", case["dtype"]])
    return case


def _tokens(case, gen):
    """Token ids of a text: a few frequent ones, a long tail, frequent ids spread over the vocabulary."""
    u = torch.rand(case["tokens"], generator=gen, device=DEVICE, dtype=torch.float64)
    rank = (torch.exp(u * math.log(case["vocab"] + 1.0)) - 1.0).floor().long().clamp(0, case["vocab"] - 1)
    ids = (rank * 7919 + 13) % case["vocab"]
    return ids.to(torch.int32 if case["ids"] == "i32" else torch.int64)


def _normal(gen, shape, dtype, std):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).mul_(std).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "lookup":
        return {"case": case, "tokens": _tokens(case, gen), "weight": _normal(gen, (case["rows"], case["width"]), dtype, 0.02)}
    if op == "lookup_grad":
        return {"case": case, "tokens": _tokens(case, gen), "grad": _normal(gen, (case["tokens"], case["width"]), dtype, 0.01)}
    if op == "quantize":
        return {"case": case, "x": _normal(gen, (case["rows"], case["width"]), dtype, 0.02)}
    if op == "int8":
        m, n, k = case["tokens"], case["out_width"], case["width"]
        state = {"case": case, "x": _normal(gen, (m, k), dtype, 1.0),
                 "values": torch.randint(-127, 128, (n, k), generator=gen, device=DEVICE, dtype=torch.int8),
                 "scales": torch.rand(n, generator=gen, device=DEVICE) * 4e-4 + 2e-4,
                 "bias": _normal(gen, (n,), torch.float32, 0.1) if case["bias"] else None}
        return state
    t, e, n, k = case["tokens"], case["experts"], case["out_width"], case["width"]
    # the router's load: a softmax of normal logits, sharper with the skew; some experts may get nothing
    load = torch.softmax(torch.randn(e, generator=gen, device=DEVICE) * case["skew"], 0)
    picks = torch.multinomial(load, t, replacement=True, generator=gen)
    sizes = torch.bincount(picks, minlength=e)
    offsets = torch.zeros(e + 1, device=DEVICE, dtype=torch.int32)
    offsets[1:] = sizes.cumsum(0)
    state = {"case": case, "offsets": offsets, "sizes": sizes.tolist(), "x": _normal(gen, (t, k), dtype, 1.0),
             "weight": _normal(gen, (e, n, k), dtype, 0.02)}
    if op == "grouped_grad":
        state["grad"] = _normal(gen, (t, n), dtype, 0.01)
    return state


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "lookup":
        local = s["tokens"].long() - case["first"]
        here = (local >= 0) & (local < case["rows"])
        rows = s["weight"][local.clamp(0, case["rows"] - 1)].float() * case["scale"]
        return torch.where(here[:, None], rows, 0.0).to(DTYPES[case["out"]])
    if op == "lookup_grad":
        local = s["tokens"].long() - case["first"]
        here = (local >= 0) & (local < case["rows"])
        total = torch.zeros(case["rows"] + 1, case["width"], device=DEVICE)  # the last row takes the other shards' tokens
        total.index_add_(0, torch.where(here, local, case["rows"]), s["grad"].float())
        return (total[:-1] * case["scale"]).to(DTYPES[case["out"]])
    if op == "quantize":
        return _to_8_bits(s["x"])
    if op == "int8":
        q, scale = _to_8_bits(s["x"])
        y = (q.float() @ s["values"].float().t()) * (scale[:, None] * s["scales"])
        return (y if s["bias"] is None else y + s["bias"]).to(s["x"].dtype)
    weights, sizes = s["weight"].float().unbind(), s["sizes"]
    if op == "grouped":
        return torch.cat([x @ w.t() for x, w in zip(s["x"].float().split(sizes), weights)]).to(s["x"].dtype)
    x, grad = s["x"].float().split(sizes), s["grad"].float().split(sizes)
    return {"rows": torch.cat([g @ w for g, w in zip(grad, weights)]).to(s["x"].dtype),
            "weight": torch.stack([g.t() @ r for g, r in zip(grad, x)]).to(DTYPES[case["out"]])}


def _to_8_bits(x):
    scale = x.abs().amax(1).float() / 127.0
    # in 64 bits: a quotient next to a half must not be rounded onto it
    q = torch.where(scale[:, None] > 0, x.double() / scale.double()[:, None], 0.0).round().clamp(-127, 127)
    return q.to(torch.int8), scale


_calls = None


def _framework():
    """The framework's functions, imported at the first call that needs them."""
    global _calls
    if _calls is None:
        from etha_amd import embedding, experts, int8

        _calls = (embedding.embedding, embedding.embedding_grad, int8.quantize_rows, int8.int8_linear, experts.grouped_linear,
                  experts.grouped_linear_grad)
    return _calls


def run(state):
    if not own:
        return _plain(state)
    embedding, embedding_grad, quantize_rows, int8_linear, grouped_linear, grouped_linear_grad = _framework()
    case = state["case"]
    op = case["op"]
    if op == "lookup":
        return embedding(state["tokens"], state["weight"], scale=case["scale"], first_row=case["first"], dtype=DTYPES[case["out"]])
    if op == "lookup_grad":
        return embedding_grad(state["grad"], state["tokens"], case["rows"], scale=case["scale"], first_row=case["first"],
                              dtype=DTYPES[case["out"]])
    if op == "quantize":
        return quantize_rows(state["x"])
    if op == "int8":
        return int8_linear(state["x"], state["values"], state["scales"], bias=state["bias"])
    if op == "grouped":
        return grouped_linear(state["x"], state["weight"], state["offsets"])
    rows, weight = grouped_linear_grad(state["grad"], state["x"], state["weight"], state["offsets"], weight_dtype=DTYPES[case["out"]])
    return {"rows": rows, "weight": weight}


def _distinct(case, n):
    """About how many different ids n tokens of _tokens() have: id r comes with probability log((r+2)/(r+1)) / log(vocab+1)."""
    total = 0.0
    lo = 0
    while lo < case["vocab"]:  # blocks of ranks that are nearly equally likely
        hi = min(case["vocab"], lo + max(1, lo // 8))
        p = math.log((hi + 1) / (lo + 1)) / math.log(case["vocab"] + 1.0) / (hi - lo)
        total += (hi - lo) * -math.expm1(n * math.log1p(-min(p, 0.999)))
        lo = hi
    return total


def work(case):
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        t, h = case["tokens"], case["width"]
        share = case["rows"] / case["vocab"]
        ids = t * (4 if case["ids"] == "i32" else 8)
        if op == "lookup":
            read = _distinct(case, t) * share * h * SIZE[case["dtype"]]
            return {"bytes": ids + read + t * h * SIZE[case["out"]], "flops": t * share * h}
        return {"bytes": ids + t * share * h * SIZE[case["dtype"]] + case["rows"] * h * SIZE[case["out"]], "flops": t * share * h}
    if op == "quantize":
        n = case["rows"] * case["width"]
        return {"bytes": n * (SIZE[case["dtype"]] + 1) + 4 * case["rows"], "flops": 3 * n}
    if op == "int8":
        m, n, k = case["tokens"], case["out_width"], case["width"]
        return {"bytes": (m * k + m * n) * SIZE[case["dtype"]] + n * k + 4 * n * (2 if case["bias"] else 1), "flops": 2 * m * n * k}
    t, e, n, k = case["tokens"], min(case["experts"], case["tokens"]), case["out_width"], case["width"]
    if op == "grouped":
        return {"bytes": 2 * (t * k + e * n * k + t * n), "flops": 2 * t * n * k}
    return {"bytes": 2 * (2 * t * k + e * n * k + t * n) + case["experts"] * n * k * SIZE[case["out"]], "flops": 4 * t * n * k}


def exact(case, seed):
    """The operators from their definitions in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        out = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device=DEVICE)
        at = torch.nonzero((s["tokens"] >= case["first"]) & (s["tokens"] < case["first"] + case["rows"])).reshape(-1)
        out[at] = s["weight"].double()[s["tokens"].long()[at] - case["first"]] * case["scale"]
        return out
    if op == "lookup_grad":
        out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device=DEVICE)
        at = torch.nonzero((s["tokens"] >= case["first"]) & (s["tokens"] < case["first"] + case["rows"])).reshape(-1)
        out.index_put_((s["tokens"].long()[at] - case["first"],), s["grad"][at].double(), accumulate=True)
        return out * case["scale"]
    if op == "quantize":
        return None, s["x"].double().abs().max(1).values / 127.0
    if op == "int8":
        x = s["x"].double()
        scale = (x.abs().max(1).values / 127.0).float().double()  # the scale is a number of 32 bits by definition
        q = torch.round(x / torch.where(scale > 0, scale, 1.0)[:, None])
        y = torch.matmul(q * scale[:, None], (s["values"].double() * s["scales"].double()[:, None]).t())
        return y if s["bias"] is None else y + s["bias"].double()
    ends = s["offsets"].tolist()
    rows = torch.zeros(case["tokens"], case["out_width"] if op == "grouped" else case["width"], dtype=torch.float64, device=DEVICE)
    weight = torch.zeros(case["experts"], case["out_width"], case["width"], dtype=torch.float64, device=DEVICE) if op == "grouped_grad" else None
    for e in range(case["experts"]):
        lo, hi = ends[e], ends[e + 1]
        w = s["weight"][e].double()
        if op == "grouped":
            rows[lo:hi] = torch.mm(s["x"][lo:hi].double(), w.t())
        else:
            g = s["grad"][lo:hi].double()
            rows[lo:hi] = torch.mm(g, w)
            weight[e] = torch.mm(g.t(), s["x"][lo:hi].double())
    return rows if op == "grouped" else {"rows": rows, "weight": weight}
