"""Projections whose weights are chosen per row, as timed cases: routing to experts, the
experts' products on MX operands, and low-rank adapters beside a shared projection.

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges;
``prepare`` / ``run`` / ``work`` say how one is set up, what one pass is and what it cannot do
without, ``exact`` what its outputs are by the operator's definition in 64 bits.  With
``own`` false ``run`` computes the operators from elementary torch operations, with ``own``
true it makes the calls of this package.

Three kinds of case:
  ``route``     logits (tokens x experts) -> experts, weights and the row plan (the pairs of a
                token and one of its experts, sorted by expert);
  ``experts``   the products of one expert layer: MX rows gathered by the plan, times each
                expert's MX matrix; ``gated`` ones hold a gate and an up projection and give
                silu(gate) * up per pair, ``summed`` ones add a token's weighted pairs up;
  ``adapters``  D = C + scale * (x A^T) B^T with one adapter (A, B) per row, or none.
"""
from __future__ import annotations

import math

import torch

own = False

EMAX = {"e4m3": 8, "e5m2": 15, "e2m1": 2}  # exponent of a format's largest binade
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _route(name, tokens, experts, top_k, **options):
    case = {"kind": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "type": "f32",
            "scoring": "softmax", "bias": False, "n_groups": 1, "top_groups": 1, "group_best": 1,
            "renormalize": True, "scale": 1.0}
    case.update(options)
    if name:
        case["name"] = name
    return case


def _experts(name, a, b, tokens, experts, top_k, n, k, **options):
    case = {"kind": "experts", "a": a, "b": b, "tokens": tokens, "experts": experts, "top_k": top_k,
            "n": n, "k": k, "pad": 0, "gated": False, "summed": False, "idle": 0, "skew": 0.0}
    case.update(options)
    if name:
        case["name"] = name
    return case


def _adapters(name, x, w, rows, adapters, rank, n, k, **options):
    case = {"kind": "adapters", "x": x, "w": w, "rows": rows, "adapters": adapters, "rank": rank,
            "n": n, "k": k, "pad": 0, "without": 0.0, "runs": False}
    case.update(options)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # The smallest call: one token of a decode step picks its experts.
        _route("route_1", 1, 64, 8),
        # A prefill batch of a model with many experts in groups: sigmoid scores, a balance bias.
        _route("route_8192_grouped", 8192, 256, 8, scoring="sigmoid", bias=True, n_groups=8, top_groups=4,
               group_best=2, scale=2.5),
        # An odd batch of 16-bit logits, whose scores tie often, over a number of experts that fills no warp.
        _route("route_1537_bf16", 1537, 60, 4, type="bf16", renormalize=False),
        # Decode, one token: its eight experts' gate and up projections, 4-bit.
        _experts("experts_1_e2m1_gated", "e2m1", "e2m1", 1, 64, 8, 1024, 4096, gated=True),
        # Decode, a batch of 32: nearly every expert is read for a few rows each.
        _experts("experts_32_e4m3_gated", "e4m3", "e4m3", 32, 64, 8, 2048, 4096, gated=True),
        # The same step's down projections, 4-bit weights under 8-bit rows, summed per token.
        _experts("experts_32_e2m1_summed", "e4m3", "e2m1", 32, 64, 8, 4096, 2048, summed=True),
        # Prefill: every expert has a few hundred rows.
        _experts("experts_2048_e4m3_gated", "e4m3", "e4m3", 2048, 32, 4, 2048, 4096, gated=True),
        # An odd batch, skewed to few experts, with padding tokens that have none.
        _experts("experts_333_ragged", "e5m2", "e5m2", 333, 7, 3, 1409, 1000, pad=24, idle=20, skew=2.0),
        # Decode, one request with its own adapter.
        _adapters("adapters_1", "bf16", "bf16", 1, 8, 16, 4096, 4096),
        # Decode, 64 requests with 64 adapters beside an up projection.
        _adapters("adapters_64", "f16", "f16", 64, 64, 16, 14336, 4096),
        # Prefill of several requests: long runs of rows with the same adapter, some without.
        _adapters("adapters_8192", "bf16", "bf16", 8192, 16, 64, 4096, 4096, runs=True, without=0.1),
        # Odd sizes and leading dimensions, f32 rows as GemmMx leaves them.
        _adapters("adapters_777_ragged", "f32", "bf16", 777, 5, 11, 1999, 1501, pad=3, without=0.2),
    ]


def _log_int(rng, lo, hi, step=1):
    """Spread over the logarithm, in multiples of `step`."""
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(x / step)) * step or step))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "experts", "adapters", "adapters"])
    if kind == "route":
        n_groups = rng.choice([1, 1, 2, 4, 8])
        experts = n_groups * rng.randint(max(2, 8 // n_groups), 256 // n_groups)
        top_groups = rng.randint(1, n_groups)
        return _route(None, _log_int(rng, 1, 8192), experts,
                      rng.randint(1, min(8, experts // n_groups * top_groups)),
                      type=rng.choice(["f32", "f32", "bf16", "f16"]), scoring=rng.choice(["softmax", "sigmoid"]),
                      bias=rng.random() < 0.5, n_groups=n_groups, top_groups=top_groups,
                      group_best=rng.choice([1, 2]), renormalize=rng.random() < 0.7,
                      scale=rng.choice([1.0, 2.5]))
    if kind == "experts":
        a, b = rng.choice([("e4m3", "e4m3"), ("e5m2", "e5m2"), ("e2m1", "e2m1"), ("e4m3", "e2m1")])
        experts = rng.randint(2, 48)
        top_k = rng.randint(1, min(8, experts))
        tokens = _log_int(rng, 1, 8192 // top_k)
        # (4-bit weights under 8-bit rows come with k in whole 128-element boxes)
        k = _log_int(rng, 256, 4096, 128 if a != b else 8)
        mode = rng.choice(["plain", "gated", "summed"])
        return _experts(None, a, b, tokens, experts, top_k, _log_int(rng, 128, 2048), k,
                        pad=-k % 32 if a == b else 0, gated=mode == "gated", summed=mode == "summed",
                        idle=rng.choice([0, 0, tokens // 8]), skew=rng.choice([0.0, 0.0, 1.5]))
    x, w = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
    rows = _log_int(rng, 1, 8192)
    grain = rng.choice([1, 8, 64])
    return _adapters(None, x, w, rows, _log_int(rng, 1, 128), _log_int(rng, 4, 64), _log_int(rng, 256, 4096, grain),
                     _log_int(rng, 256, 4096, grain), pad=rng.choice([0, 0, 3]),
                     without=rng.choice([0.0, 0.0, 0.3]), runs=rng.random() < 0.5)


# ---- operands ---------------------------------------------------------------------------


def _quantise(x, fmt):
    """Rows of f32 values (last dimension a multiple of 32) as MX elements and E8M0 scales: the
    largest of each 32 falls in the format's top binade."""
    blocks = x.unflatten(-1, (-1, 32))
    exponent = torch.frexp(blocks.abs().amax(-1).clamp_min(2.0 ** -60))[1] - 1 - EMAX[fmt]
    y = torch.ldexp(blocks, -exponent.unsqueeze(-1)).flatten(-2)
    scales = (exponent + 127).to(torch.uint8)
    if fmt == "e4m3":
        return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scales
    if fmt == "e5m2":
        return y.clamp(-57344, 57344).to(torch.float8_e5m2).view(torch.uint8), scales
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    code = torch.bucketize(y.abs(), edges).to(torch.uint8) | ((y < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4), scales


def _plan(ids, experts):
    """Pairs sorted by expert (stable), and where each expert's run starts."""
    flat = ids.flatten().long()
    valid = (flat >= 0) & (flat < experts)
    key = torch.where(valid, flat, torch.full_like(flat, experts))
    order = torch.sort(key, stable=True)[1].int()
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = counts.cumsum(0)
    place = torch.arange(order.numel(), device=ids.device)
    return offsets, torch.where(place < offsets[-1], order, torch.full_like(order, -1))


def _prepare_route(case, g, dev):
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    state = {"logits": (2.0 * torch.randn((t, e), device=dev, generator=g)).to(FLOAT[case["type"]]),
             "bias": 0.1 * torch.randn((e,), device=dev, generator=g) if case["bias"] else None,
             "ids": torch.zeros((t, k), dtype=torch.int32, device=dev),
             "weights": torch.zeros((t, k), dtype=torch.float32, device=dev),
             "offsets": torch.zeros((e + 1,), dtype=torch.int32, device=dev),
             "order": torch.zeros((t * k,), dtype=torch.int32, device=dev)}
    state["out"] = {name: state[name] for name in ("ids", "weights", "offsets", "order")}
    return state


def _call_route(case, state):
    import cpu_ops_b200 as c
    op = c.RouteExperts(_storage(case["type"]), stream=torch.cuda.current_stream().cuda_stream, asynchronous=True)
    return op, op.Arguments(
        c.RouteCoord(case["tokens"], case["experts"], case["top_k"]), c.TensorRef(state["logits"], case["experts"]),
        state["ids"], state["weights"], c.RowPlan(state["offsets"], state["order"]),
        c.Scoring.kSigmoid if case["scoring"] == "sigmoid" else c.Scoring.kSoftmax, state["bias"],
        c.ExpertGroups(case["n_groups"], case["top_groups"], case["group_best"]),
        case["renormalize"], case["scale"])


def _prepare_experts(case, g, dev):
    t, e, top_k, n, k = case["tokens"], case["experts"], case["top_k"], case["n"], case["k"]
    rows = t * top_k
    lead = k + case["pad"]                     # elements from one row to the next
    wide = (lead + 31) // 32 * 32              # (the operands are made with whole blocks of 32)
    per_byte_a, per_byte_b = (2 if case[s] == "e2m1" else 1 for s in "ab")
    # a token's experts: distinct, the first ones likelier where the batch is skewed
    score = torch.rand((t, e), device=dev, generator=g).log() / torch.exp(
        -case["skew"] * torch.arange(e, device=dev) / max(1, e - 1))
    ids = score.topk(top_k, dim=1)[1].int().contiguous()
    if case["idle"]:
        ids[t - case["idle"]:] = -1            # padding tokens at the end of the batch
    pair_weights = torch.rand((t, top_k), device=dev, generator=g) + 0.05
    pair_weights = pair_weights / pair_weights.sum(1, keepdim=True)
    offsets, order = _plan(ids, e)

    def matrix(count, fmt, sigma):
        x = torch.randn((count, wide), device=dev, generator=g) * sigma
        x[:, k:] = 0
        return _quantise(x, fmt)

    # the first product reads a row per token, the one that sums reads a row per pair
    a_rows = rows if case["summed"] else t
    A, SA = matrix(a_rows, case["a"], 1.0)
    n_b = 2 * n if case["gated"] else n
    B = torch.empty((e, n_b, wide // per_byte_b), dtype=torch.uint8, device=dev)
    SB = torch.empty((e, n_b, wide // 32), dtype=torch.uint8, device=dev)
    for i in range(e):
        B[i], SB[i] = matrix(n_b, case["b"], 1.0 / math.sqrt(k))
    A, B = A[:, :lead // per_byte_a].contiguous(), B[..., :lead // per_byte_b].contiguous()
    D = torch.zeros((t if case["summed"] else rows, n), dtype=torch.float32, device=dev)
    return {"A": A, "SA": SA, "B": B, "SB": SB, "ids": ids, "weights": pair_weights, "offsets": offsets,
            "order": order, "D": D, "out": D, "ends": offsets.tolist()}


def _call_experts(case, state):
    import cpu_ops_b200 as c
    top_k, n, k, lead = case["top_k"], case["n"], case["k"], case["k"] + case["pad"]
    groups = (lead + 31) // 32
    summed = case["summed"]
    op = c.GemmMxGrouped(_storage(case["a"]), _storage(case["b"]), gated=case["gated"],
                         stream=torch.cuda.current_stream().cuda_stream, asynchronous=True)
    return op, op.Arguments(
        c.GroupedCoord(case["tokens"] * top_k, n, k, case["experts"]),
        c.MxTensorRef(state["A"], state["SA"], lead, groups), c.MxTensorRef(state["B"], state["SB"], lead, groups),
        c.RowPlan(state["offsets"], state["order"]), c.TensorRef(state["D"], n),
        pairs_per_a_row=1 if summed else top_k, row_weights=state["weights"] if summed else None,
        pairs_per_d_row=top_k if summed else 1, ids=state["ids"] if summed else None)


def _prepare_adapters(case, g, dev):
    m, count, r, n, k, pad = (case[s] for s in ("rows", "adapters", "rank", "n", "k", "pad"))
    x = torch.randn((m, k + pad), device=dev, generator=g).to(FLOAT[case["x"]])
    A = (torch.randn((count, r, k + pad), device=dev, generator=g) / math.sqrt(k)).to(FLOAT[case["w"]])
    B = (torch.randn((count, n, r + pad), device=dev, generator=g) / math.sqrt(r)).to(FLOAT[case["w"]])
    scales = torch.rand((count,), device=dev, generator=g) + 0.5
    if case["runs"]:   # requests of different lengths, one after another
        ends = torch.rand((count,), device=dev, generator=g).cumsum(0)
        place = torch.arange(m, device=dev) * (ends[-1] / m)
        ids = torch.searchsorted(ends, place).clamp_max(count - 1)
    else:
        ids = torch.randint(0, count, (m,), device=dev, generator=g)
    none = torch.rand((m,), device=dev, generator=g) < case["without"]
    ids = torch.where(none, torch.full_like(ids, -1), ids).int()
    C = torch.randn((m, n + pad), device=dev, generator=g)
    # (D apart from C, the shared projection's result, so that every pass gives the same)
    D = torch.zeros_like(C)
    return {"x": x, "A": A, "B": B, "scales": scales, "ids": ids, "C": C, "D": D, "out": D[:, :n],
            "runs": _runs(ids, count)}


def _call_adapters(case, state):
    import cpu_ops_b200 as c
    m, count, r, n, k, pad = (case[s] for s in ("rows", "adapters", "rank", "n", "k", "pad"))
    op = c.LowRankAdapters(_storage(case["x"]), _storage(case["w"]),
                           stream=torch.cuda.current_stream().cuda_stream, asynchronous=True)
    return op, op.Arguments(
        c.AdapterCoord(m, n, k, r, count), c.TensorRef(state["x"], k + pad),
        c.AdapterRef(state["A"], k + pad, r * (k + pad)), c.AdapterRef(state["B"], r + pad, n * (r + pad)),
        state["ids"], c.TensorRef(state["C"], n + pad), c.TensorRef(state["D"], n + pad), state["scales"])


def _runs(ids, count):
    """(adapter, its rows) for each adapter in use: what a program without the operator sorts out
    once per batch."""
    return [(i, rows) for i in range(count) if (rows := (ids == i).nonzero().flatten()).numel()]


def _storage(name):
    import cpu_ops_b200 as c
    return {"e4m3": c.fp8e4m3_t, "e5m2": c.fp8e5m2_t, "e2m1": c.fp4e2m1_t,
            "f32": c.f32_t, "f16": c.f16_t, "bf16": c.bf16_t}[name]


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    make = {"route": _prepare_route, "experts": _prepare_experts, "adapters": _prepare_adapters}[case["kind"]]
    state = make(case, g, dev)
    state["case"] = case
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        call = {"route": _call_route, "experts": _call_experts, "adapters": _call_adapters}[case["kind"]]
        op, args = call(case, state)
        state["issue"], state["call"] = op.run, op.describe(args)
    return state


# ---- one pass -----------------------------------------------------------------------------


def run(state):
    if own:
        import cpu_ops_b200 as c
        if state["issue"](state["call"]) != c.Status.kSuccess:
            raise RuntimeError(c._capi.last_error())
        return state["out"]
    plain = {"route": _plain_route, "experts": _plain_experts, "adapters": _plain_adapters}
    return plain[state["case"]["kind"]](state)


def _plain_route(state):
    # In 64 bits: two experts whose scores differ in the ninth digit have to come out in order.
    case, x = state["case"], state["logits"].double()
    t, e = x.shape
    if case["scoring"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True))
        score = p / p.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score + state["bias"].double() if case["bias"] else score
    if case["n_groups"] > 1:
        grouped = choice.view(t, case["n_groups"], -1)
        best = grouped.sort(dim=2, descending=True)[0][..., :case["group_best"]].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(keep.unsqueeze(2), grouped, torch.full_like(grouped, -math.inf)).view(t, e)
    ids = choice.sort(dim=1, descending=True, stable=True)[1][:, :case["top_k"]]
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    offsets, order = _plan(ids, e)
    return {"ids": ids.int(), "weights": (weights * case["scale"]).float(), "offsets": offsets, "order": order}


def _values(codes, scales, fmt, k):
    """MX elements as f32 numbers."""
    if fmt == "e2m1":
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
        x = table[torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).int()]
    else:
        x = codes.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.float8_e5m2).float()
    x = x[..., :k]
    factor = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127)
    return x * factor.repeat_interleave(32, dim=-1)[..., :k]


def _plain_experts(state):
    case, D = state["case"], state["D"]
    n, k, top_k = case["n"], case["k"], case["top_k"]
    A = _values(state["A"], state["SA"], case["a"], k)
    pairs = torch.zeros((state["order"].numel(), n), dtype=torch.float32, device=D.device) if case["summed"] else D
    ends = state["ends"]
    for i in range(case["experts"]):
        if ends[i] == ends[i + 1]:
            continue
        q = state["order"][ends[i]:ends[i + 1]].long()
        y = A[q if case["summed"] else q // top_k] @ _values(state["B"][i], state["SB"][i], case["b"], k).t()
        if case["gated"]:
            gate, up = y[:, :n], y[:, n:]
            y = gate / (1.0 + torch.exp(-gate)) * up
        if case["summed"]:
            y = y * state["weights"].flatten()[q].unsqueeze(1)
        pairs[q] = y
    if case["summed"]:
        torch.sum(pairs.view(case["tokens"], top_k, n), 1, out=D)
    return D


def _plain_adapters(state):
    D, C = state["D"], state["C"]
    D.copy_(C)
    n, k, r = (state["case"][s] for s in ("n", "k", "rank"))
    for i, rows in state["runs"]:
        u = state["x"][rows, :k].float() @ state["A"][i, :, :k].float().t()
        y = u @ state["B"][i, :, :r].float().t()
        D[rows, :n] += y * state["scales"][i]
    return D[:, :n]


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    if case["kind"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": t * e * size + (4 * e if case["bias"] else 0) + t * k * 12 + 4 * (e + 1),
                "flops": 5.0 * t * e}
    if case["kind"] == "experts":
        t, e, top_k, n, k = (case[s] for s in ("tokens", "experts", "top_k", "n", "k"))
        live = t - case["idle"]
        bits = {"e2m1": 4.25, "e4m3": 8.25, "e5m2": 8.25}  # with the share of a block's scale
        n_b = 2 * n if case["gated"] else n
        # experts that no row goes to are not read: their expected number, were all equally likely
        busy = e * (1.0 - (1.0 - top_k / e) ** live)
        a_rows = live * top_k if case["summed"] else live
        d_rows = t if case["summed"] else live * top_k
        return {"bytes": (a_rows * bits[case["a"]] + busy * n_b * bits[case["b"]]) * k / 8 + d_rows * n * 4
                + live * top_k * 4, "flops": 2.0 * live * top_k * n_b * k}
    m, count, r, n, k = (case[s] for s in ("rows", "adapters", "rank", "n", "k"))
    live = m * (1.0 - case["without"])
    busy = count * (1.0 - (1.0 - 1.0 / count) ** live)
    sizes = {"f32": 4, "f16": 2, "bf16": 2}
    return {"bytes": live * k * sizes[case["x"]] + busy * r * (n + k) * sizes[case["w"]]
            + 8 * n * m, "flops": 2.0 * live * r * (n + k)}


# ---- the operators by their definition, in 64 bits ---------------------------------------------


def exact(case, seed):
    # Nearly all of it is matrix products in 64 bits, at some 20e12 operations a second.
    if work(case)["flops"] > 3.2e11:
        return None
    state = _inputs(case, seed)
    return {"route": _exact_route, "experts": _exact_experts, "adapters": _exact_adapters}[case["kind"]](case, state)


def _exact_route(case, state):
    x = state["logits"].cpu().double()
    t, e = x.shape
    top_k, per = case["top_k"], e // case["n_groups"]
    if case["scoring"] == "softmax":
        score = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
    else:
        score = torch.where(x >= 0, 1 / (1 + torch.exp(-x)), torch.exp(x) / (1 + torch.exp(x)))
    choice = score + (state["bias"].cpu().double() if case["bias"] else 0.0)
    if case["scoring"] == "softmax" and not case["bias"]:
        rank_by = x       # the scores' order is the logits' own
    else:
        rank_by = choice
    if case["n_groups"] > 1:
        parts = [choice[:, i * per:(i + 1) * per] for i in range(case["n_groups"])]
        best = torch.stack([p.topk(min(case["group_best"], per), dim=1)[0].sum(1) for p in parts], 1)
        # a group's place: how many come before it
        ahead = (best.unsqueeze(1) > best.unsqueeze(2)).sum(2)
        index = torch.arange(case["n_groups"])
        ahead += ((best.unsqueeze(1) == best.unsqueeze(2)) & (index.view(1, 1, -1) < index.view(1, -1, 1))).sum(2)
        out = (ahead >= case["top_groups"]).repeat_interleave(per, 1)
        rank_by = rank_by.masked_fill(out, -math.inf)
    ids = torch.empty((t, top_k), dtype=torch.int64)
    left = rank_by.clone()
    for j in range(top_k):
        best = left.amax(1, keepdim=True)
        ids[:, j] = (left == best).int().argmax(1)   # the first of those that are equal
        left.scatter_(1, ids[:, j:j + 1], -math.inf)
    weights = score.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True)
    members = [(ids.flatten() == i).nonzero().flatten() for i in range(e)]
    offsets = torch.tensor([0] + [m.numel() for m in members]).cumsum(0)
    return {"ids": ids.int(), "weights": weights * case["scale"], "offsets": offsets.int(),
            "order": torch.cat(members).int()}


def _decode(codes, scales, fmt, k):
    """MX elements in 64 bits, from their sign, exponent and fraction fields."""
    if fmt == "e2m1":
        codes = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    mantissa, bits, bias = {"e4m3": (3, 4, 7), "e5m2": (2, 5, 15), "e2m1": (1, 2, 1)}[fmt]
    v = codes[..., :k].int()
    field = (v >> mantissa) & ((1 << bits) - 1)
    fraction = (v & ((1 << mantissa) - 1)).double() / (1 << mantissa)
    size = torch.ldexp(fraction + (field > 0), field.clamp_min(1) - bias)
    sign = 1 - 2 * ((v >> (mantissa + bits)) & 1)
    block = torch.arange(k, device=codes.device) // 32
    return torch.ldexp(sign * size, scales[..., block].int() - 127)


def _exact_experts(case, state):
    n, k, top_k = case["n"], case["k"], case["top_k"]
    A = _decode(state["A"], state["SA"], case["a"], k)
    ids = state["ids"].flatten()
    y = torch.zeros((ids.numel(), n), dtype=torch.float64, device=A.device)
    token = torch.arange(ids.numel(), device=A.device) // top_k
    for i in range(case["experts"]):
        mine = (ids == i).nonzero().flatten()
        if mine.numel() == 0:
            continue
        w = _decode(state["B"][i], state["SB"][i], case["b"], k)
        x = A[mine] if case["summed"] else A[token[mine]]
        if case["gated"]:
            y[mine] = torch.nn.functional.silu(x @ w[:n].t()) * (x @ w[n:].t())
        else:
            y[mine] = x @ w.t()
    if case["summed"]:
        y = torch.einsum("tsn,ts->tn", y.view(-1, top_k, n), state["weights"].double())
    return y


def _exact_adapters(case, state):
    m, count, r, n, k = (case[s] for s in ("rows", "adapters", "rank", "n", "k"))
    x = state["x"][:, :k].double()
    out = state["C"][:, :n].double().clone()
    for i in range(count):
        mine = (state["ids"] == i).nonzero().flatten()
        if mine.numel():
            product = state["B"][i, :, :r].double() @ (state["A"][i, :, :k].double() @ x[mine].t())
            out[mine] += float(state["scales"][i]) * product.t()
    return out
