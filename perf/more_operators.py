"""Training operators of 16-bit layers beside the quantised products, as timed cases: the product of
16-bit matrices with bias, activation and residual in its epilogue, that epilogue's gradient, layer
norm and its gradient, and the balance loss of a router with counts and gradient.

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges;
``prepare`` / ``run`` / ``work`` say how one is set up, what one pass is and what it cannot do
without, ``exact`` what its outputs are by the operator's definition in 64 bits.  With
``own`` false ``run`` computes the operators from elementary torch operations, with ``own``
true it makes the calls of this package.

Five kinds of case:
  ``product``    D = act(A B + bias) + C, and z = A B + bias where a backward pass will need it;
                 A and B row- or column-major, so that the products of a backward pass are cases too;
  ``epilogue``   dz = dy * act'(z) and dbias = the column sums of dz;
  ``norm``       y = (x - mean) * rstd * gamma + beta, row by row, with mean and rstd;
  ``norm_grad``  dx (plus a residual's gradient), dgamma and dbeta of that;
  ``balance``    counts per expert, loss = c * experts * sum_e f_e P_e of the experts' shares f of the
                 pairs and their mean scores P, and the loss's gradient by the logits.
"""
from __future__ import annotations

import math

import torch

own = False

FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GELU_C, GELU_A = math.sqrt(2.0 / math.pi), 0.044715
EPS = 1e-5


def _case(kind, name, options, **defaults):
    case = {"kind": kind}
    case.update(defaults)
    case.update(options)
    if name:
        case["name"] = name
    return case


def _product(name, m, n, k, **options):
    # a, b: whether A (m x k) and B (k x n) are stored by rows or by columns
    return _case("product", name, options, m=m, n=n, k=k, type="bf16", d="bf16", a="row", b="col", bias=True, act="none",
                 residual=False, z=False, pad=0)


def _epilogue(name, m, n, **options):
    return _case("epilogue", name, options, m=m, n=n, type="bf16", act="gelu", pad=0)


def _norm(name, m, n, **options):
    return _case("norm", name, options, m=m, n=n, x="bf16", y="bf16", pad=0)


def _norm_grad(name, m, n, **options):
    return _case("norm_grad", name, options, m=m, n=n, x="bf16", y="bf16", residual=False, pad=0)


def _balance(name, tokens, experts, top_k, **options):
    return _case("balance", name, options, tokens=tokens, experts=experts, top_k=top_k, type="f32", scoring="softmax",
                 idle=0, pad=0)


def listed():
    return [
        # Decode: a batch of eight tokens through an up projection; reading the weights is all of it.
        _product("product_8", 8, 14336, 4096, act="silu"),
        # Training, forward: the projection that ends a block and adds to the residual stream.
        _product("product_8192_residual", 8192, 4096, 4096, residual=True),
        # Training, backward: a weight's gradient, added to what earlier micro-batches left, in f32.
        _product("product_weight_gradient", 4096, 2048, 8192, a="col", b="row", d="f32", bias=False, residual=True),
        # Odd sizes and leading dimensions, weights by rows, z kept for the backward pass.
        _product("product_777_ragged", 777, 1999, 1501, type="f16", d="f16", b="row", act="gelu", residual=True, z=True,
                 pad=3),
        # Training: the activation between a feed-forward layer's two projections.
        _epilogue("epilogue_8192", 8192, 14336),
        # An odd batch.
        _epilogue("epilogue_777_ragged", 777, 1409, type="f16", act="silu", pad=3),
        # Decode: eight tokens of an f32 residual stream on their way to a 16-bit projection.
        _norm("norm_8", 8, 4096, x="f32"),
        # Training or prefill.
        _norm("norm_8192", 8192, 4096),
        # Training, with the gradient that comes past the norm on the residual stream.
        _norm_grad("norm_grad_8192", 8192, 4096, residual=True),
        # Odd sizes, an f32 residual stream under a 16-bit layer.
        _norm_grad("norm_grad_777_ragged", 777, 1999, x="f32", y="f16", pad=3),
        # A batch of a model with many experts and sigmoid scores.
        _balance("balance_8192", 8192, 256, 8, scoring="sigmoid"),
        # An odd batch of 16-bit logits with padding tokens at its end.
        _balance("balance_1537_bf16", 1537, 60, 4, type="bf16", idle=100),
    ]


def _log_int(rng, lo, hi, step=1):
    """Spread over the logarithm, in multiples of `step`."""
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(x / step)) * step or step))


def draw(rng):
    kind = rng.choice(["product", "product", "product", "epilogue", "norm", "norm_grad", "balance"])
    if kind == "product":
        kind16 = rng.choice(["bf16", "f16"])
        # forward (weights by rows or columns), the gradient of its input, the gradient of its weights
        way = rng.choice(["forward", "forward", "forward", "input", "weight"])
        grain = rng.choice([1, 8, 64])
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 128, 8192, grain), _log_int(rng, 128, 8192, grain)
        if way == "weight":
            m, n, k = n, _log_int(rng, 128, 4096, grain), max(16, m)
        most = 8192 * 4096 * 4096
        if m * n * k > most:
            k = max(128, most // (m * n) // 64 * 64)
        pad = rng.choice([0, 0, 0, 8, 3])
        if way == "input":
            return _product(None, m, n, k, type=kind16, d=kind16, b="row", bias=False, pad=pad)
        if way == "weight":
            return _product(None, m, n, k, type=kind16, d=rng.choice(["f32", "f32", kind16]), a="col", b="row", bias=False,
                            residual=rng.random() < 0.5, pad=pad)
        act = rng.choice(["none", "relu", "gelu", "silu"])
        return _product(None, m, n, k, type=kind16, d=rng.choice([kind16, kind16, "f32"]), b=rng.choice(["col", "col", "row"]),
                        bias=rng.random() < 0.7, act=act, residual=rng.random() < 0.4,
                        z=act != "none" and rng.random() < 0.5, pad=pad)
    if kind == "epilogue":
        kind = rng.choice(["bf16", "bf16", "f16", "f32"])
        m, n = _log_int(rng, 1, 8192), _log_int(rng, 64, 14336, rng.choice([1, 8]))
        m = min(m, 2 * 8192 * 14336 // (n * SIZE[kind]))
        return _epilogue(None, m, n, type=kind, act=rng.choice(["none", "relu", "gelu", "silu"]), pad=rng.choice([0, 0, 8, 3]))
    if kind in ("norm", "norm_grad"):
        x, y = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16"), ("f32", "f16")])
        m, n = _log_int(rng, 1, 8192), _log_int(rng, 64, 8192, rng.choice([1, 8]))
        m = min(m, 8192 * 4096 // n)
        pad = rng.choice([0, 0, 8, 3])
        if kind == "norm":
            return _norm(None, m, n, x=x, y=y, pad=pad)
        return _norm_grad(None, m, n, x=x, y=y, residual=rng.random() < 0.5, pad=pad)
    tokens, experts = _log_int(rng, 1, 8192), rng.randint(4, 256)
    return _balance(None, tokens, experts, rng.randint(1, min(8, experts)), type=rng.choice(["f32", "f32", "bf16", "f16"]),
                    scoring=rng.choice(["softmax", "sigmoid"]), idle=rng.choice([0, 0, tokens // 8]),
                    pad=rng.choice([0, 0, 3]))


# ---- operands ---------------------------------------------------------------------------


def _matrix(g, dev, rows, cols, pad, kind, sigma=1.0, offset=0.0):
    """`rows` rows of `cols`, `cols + pad` elements apart."""
    x = torch.randn((rows, cols + pad), device=dev, generator=g)
    if sigma != 1.0 or offset:
        x = x * sigma + offset
    return x.to(FLOAT[kind])


def _prepare_product(case, g, dev):
    m, n, k, pad, kind = (case[s] for s in ("m", "n", "k", "pad", "type"))
    state = {"A": _matrix(g, dev, m, k, pad, kind) if case["a"] == "row" else _matrix(g, dev, k, m, pad, kind),
             "B": (_matrix(g, dev, k, n, pad, kind, k ** -0.5) if case["b"] == "row"
                   else _matrix(g, dev, n, k, pad, kind, k ** -0.5)),
             "bias": 0.2 * torch.randn((n,), device=dev, generator=g) if case["bias"] else None,
             "C": _matrix(g, dev, m, n, pad, case["d"]) if case["residual"] else None,
             "D": torch.zeros((m, n + pad), dtype=FLOAT[case["d"]], device=dev),
             "Z": torch.zeros((m, n + pad), dtype=FLOAT[case["d"]], device=dev) if case["z"] else None}
    state["out"] = {s: state[s][:, :n] for s in ("D", "Z") if state[s] is not None}
    return state


def _prepare_epilogue(case, g, dev):
    m, n, pad, kind = (case[s] for s in ("m", "n", "pad", "type"))
    state = {"dY": _matrix(g, dev, m, n, pad, kind, 0.1), "Z": _matrix(g, dev, m, n, pad, kind, 1.5),
             "dZ": torch.zeros((m, n + pad), dtype=FLOAT[kind], device=dev),
             "dbias": torch.zeros((n,), dtype=torch.float32, device=dev)}
    state["out"] = {"dZ": state["dZ"][:, :n], "dbias": state["dbias"]}
    return state


def _prepare_norm(case, g, dev):
    m, n, pad = (case[s] for s in ("m", "n", "pad"))
    state = {"X": _matrix(g, dev, m, n, pad, case["x"], 2.0, 0.5),
             "gamma": 1.0 + 0.2 * torch.randn((n,), device=dev, generator=g),
             "beta": 0.2 * torch.randn((n,), device=dev, generator=g),
             "Y": torch.zeros((m, n + pad), dtype=FLOAT[case["y"]], device=dev),
             "mean": torch.zeros((m,), dtype=torch.float32, device=dev),
             "rstd": torch.zeros((m,), dtype=torch.float32, device=dev)}
    state["out"] = {"Y": state["Y"][:, :n], "mean": state["mean"], "rstd": state["rstd"]}
    return state


def _prepare_norm_grad(case, g, dev):
    m, n, pad = (case[s] for s in ("m", "n", "pad"))
    state = {"X": _matrix(g, dev, m, n, pad, case["x"], 2.0, 0.5), "dY": _matrix(g, dev, m, n, pad, case["y"], 0.1),
             "dR": _matrix(g, dev, m, n, pad, case["x"], 0.1) if case["residual"] else None,
             "gamma": 1.0 + 0.2 * torch.randn((n,), device=dev, generator=g),
             "dX": torch.zeros((m, n + pad), dtype=FLOAT[case["x"]], device=dev),
             "dgamma": torch.zeros((n,), dtype=torch.float32, device=dev),
             "dbeta": torch.zeros((n,), dtype=torch.float32, device=dev)}
    x = state["X"][:, :n].float()   # what the forward pass left
    mean = x.mean(1)
    var = (x - mean.unsqueeze(1)).square().mean(1)
    state["mean"], state["rstd"] = mean, 1.0 / torch.sqrt(var + EPS)
    state["out"] = {"dX": state["dX"][:, :n], "dgamma": state["dgamma"], "dbeta": state["dbeta"]}
    return state


def _prepare_balance(case, g, dev):
    t, e, top_k, pad = (case[s] for s in ("tokens", "experts", "top_k", "pad"))
    # (some experts are liked better than others, which is what the loss is there for)
    logits = 1.5 * torch.randn((t, e + pad), device=dev, generator=g) + 0.5 * torch.randn((e + pad,), device=dev, generator=g)
    logits = logits.to(FLOAT[case["type"]])
    ids = logits[:, :e].float().topk(top_k, dim=1)[1].int().contiguous()
    if case["idle"]:
        ids[t - case["idle"]:] = -1   # padding tokens at the end of the batch
    state = {"logits": logits, "ids": ids, "counts": torch.zeros((e,), dtype=torch.int32, device=dev),
             "loss": torch.zeros((1,), dtype=torch.float32, device=dev),
             "upstream": 0.5 + torch.rand((1,), device=dev, generator=g), "dlogits": torch.zeros_like(logits)}
    state["out"] = {"counts": state["counts"], "loss": state["loss"], "dlogits": state["dlogits"][:, :e]}
    return state


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    make = {"product": _prepare_product, "epilogue": _prepare_epilogue, "norm": _prepare_norm,
            "norm_grad": _prepare_norm_grad, "balance": _prepare_balance}[case["kind"]]
    state = make(case, g, dev)
    state["case"] = case
    return state


def prepare(case, seed):
    return _inputs(case, seed)


# ---- one pass -----------------------------------------------------------------------------


def run(state):
    if own:
        import cpu_ops_b200 as c
        stream = torch.cuda.current_stream().cuda_stream
        if state.get("stream") != stream:   # a program that repeats a call keeps its descriptor
            call = {"product": _call_product, "epilogue": _call_epilogue, "norm": _call_norm,
                    "norm_grad": _call_norm_grad, "balance": _call_balance}[state["case"]["kind"]]
            op, args = call(state["case"], state, {"stream": stream, "asynchronous": True})
            state["stream"], state["issue"], state["call"] = stream, op.run, op.describe(args)
        if state["issue"](state["call"]) != c.Status.kSuccess:
            raise RuntimeError(c._capi.last_error())
        return state["out"]
    plain = {"product": _plain_product, "epilogue": _plain_epilogue, "norm": _plain_norm, "norm_grad": _plain_norm_grad,
             "balance": _plain_balance}
    return plain[state["case"]["kind"]](state)


def _storage(name):
    import cpu_ops_b200 as c
    return {"f32": c.f32_t, "f16": c.f16_t, "bf16": c.bf16_t}[name]


def _activation(name):
    import cpu_ops_b200 as c
    return {"none": None, "relu": c.Relu(), "gelu": c.Gelu(), "silu": c.Silu()}[name]


def _ref(buffer):
    import cpu_ops_b200 as c
    return c.TensorRef() if buffer is None else c.TensorRef(buffer, buffer.shape[1])


def _call_product(case, state, place):
    import cpu_ops_b200 as c
    layout = {"row": c.RowMajor, "col": c.ColumnMajor}
    op = {"bf16": c.GemmBF16, "f16": c.GemmF16}[case["type"]](layout[case["a"]], layout[case["b"]],
                                                             storage_d=_storage(case["d"]), **place)
    return op, op.Arguments(
        c.GemmCoord(case["m"], case["n"], case["k"]), _ref(state["A"]), _ref(state["B"]), _ref(state["C"]), _ref(state["D"]),
        c.BiasActivation(state["bias"], _activation(case["act"]), beta=1.0 if case["residual"] else 0.0),
        ref_Z=_ref(state["Z"]))


def _call_epilogue(case, state, place):
    import cpu_ops_b200 as c
    op = c.BiasActivationGrad(_storage(case["type"]), _activation(case["act"]), **place)
    return op, op.Arguments(c.RowsCoord(case["m"], case["n"]), _ref(state["dY"]), _ref(state["Z"]), _ref(state["dZ"]),
                            state["dbias"])


def _call_norm(case, state, place):
    import cpu_ops_b200 as c
    op = c.LayerNorm(_storage(case["x"]), _storage(case["y"]), **place)
    return op, op.Arguments(c.RowsCoord(case["m"], case["n"]), _ref(state["X"]), state["gamma"], state["beta"],
                            _ref(state["Y"]), state["mean"], state["rstd"], EPS)


def _call_norm_grad(case, state, place):
    import cpu_ops_b200 as c
    op = c.LayerNormGrad(_storage(case["x"]), _storage(case["y"]), **place)
    return op, op.Arguments(c.RowsCoord(case["m"], case["n"]), _ref(state["dY"]), _ref(state["X"]), state["gamma"],
                            state["mean"], state["rstd"], _ref(state["dX"]), state["dgamma"], state["dbeta"],
                            ref_dR=_ref(state["dR"]))


def _call_balance(case, state, place):
    import cpu_ops_b200 as c
    op = c.BalanceLoss(_storage(case["type"]), **place)
    return op, op.Arguments(
        c.RouteCoord(case["tokens"], case["experts"], case["top_k"]), _ref(state["logits"]), state["ids"], state["counts"],
        state["loss"], _ref(state["dlogits"]), c.Scoring.kSigmoid if case["scoring"] == "sigmoid" else c.Scoring.kSoftmax,
        0.01, state["upstream"])


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.tanh(GELU_C * (z + GELU_A * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain_product(state):
    case = state["case"]
    m, n, k = case["m"], case["n"], case["k"]
    a = state["A"][:, :k].float() if case["a"] == "row" else state["A"][:, :m].float().t()
    b = state["B"][:, :n].float() if case["b"] == "row" else state["B"][:, :k].float().t()
    z = a @ b
    if case["bias"]:
        z = z + state["bias"]
    d = _plain_act(z, case["act"])
    if case["residual"]:
        d = d + state["C"][:, :n].float()
    out = {"D": d.to(FLOAT[case["d"]])}
    if case["z"]:
        out["Z"] = z.to(FLOAT[case["d"]])
    return out


def _plain_epilogue(state):
    case = state["case"]
    n = case["n"]
    dy, z = state["dY"][:, :n].float(), state["Z"][:, :n].float()
    if case["act"] == "relu":
        dz = torch.where(z <= 0, torch.zeros_like(dy), dy)
    elif case["act"] == "gelu":
        t = torch.tanh(GELU_C * (z + GELU_A * z * z * z))
        dz = dy * (0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * (GELU_C * (1.0 + 3.0 * GELU_A * z * z)))
    elif case["act"] == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        dz = dy * (s * (1.0 + z * (1.0 - s)))
    else:
        dz = dy
    return {"dZ": dz.to(FLOAT[case["type"]]), "dbias": dz.sum(0)}


def _plain_norm(state):
    case = state["case"]
    x = state["X"][:, :case["n"]].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    y = d * rstd * state["gamma"] + state["beta"]
    return {"Y": y.to(FLOAT[case["y"]]), "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _plain_norm_grad(state):
    case = state["case"]
    n = case["n"]
    dy, rstd = state["dY"][:, :n].float(), state["rstd"].unsqueeze(1)
    xhat = (state["X"][:, :n].float() - state["mean"].unsqueeze(1)) * rstd
    g = dy * state["gamma"]
    dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    if case["residual"]:
        dx = dx + state["dR"][:, :n].float()
    return {"dX": dx.to(FLOAT[case["x"]]), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}


def _plain_balance(state):
    case = state["case"]
    t, e = case["tokens"], case["experts"]
    ids = state["ids"].long()
    valid = (ids >= 0) & (ids < e)
    counts = torch.bincount(torch.where(valid, ids, torch.full_like(ids, e)).flatten(), minlength=e + 1)[:e]
    live = valid.any(1, keepdim=True).float()
    tokens = live.sum()
    # the shares as differences from 1 / e, in 64 bits: what the gradient is made of
    share = (counts.double() / counts.sum() - 1.0 / e).float()
    x = state["logits"][:, :e].float()
    if case["scoring"] == "softmax":
        p = torch.exp(x - x.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
        slope = p
    else:
        s = 1.0 / (1.0 + torch.exp(-x))
        p = s / s.sum(1, keepdim=True)
        slope = p * (1.0 / (1.0 + torch.exp(x)))
    mean_score = (p * live).sum(0) / tokens
    loss = 0.01 * (1.0 + e * (share * mean_score).sum())
    gradient = slope * (share - (p * share).sum(1, keepdim=True)) * live * (state["upstream"] * 0.01 * e / tokens)
    return {"counts": counts.int(), "loss": loss.reshape(1), "dlogits": gradient.to(FLOAT[case["type"]])}


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "product":
        m, n, k, size = case["m"], case["n"], case["k"], SIZE[case["d"]]
        return {"bytes": 2 * k * (m + n) + (4 * n if case["bias"] else 0) + m * n * size * (1 + case["residual"] + case["z"]),
                "flops": 2.0 * m * n * k}
    if kind == "balance":
        t, e, top_k = case["tokens"], case["experts"], case["top_k"]
        live = t - case["idle"]
        return {"bytes": (live + t) * e * SIZE[case["type"]] + 4 * t * top_k + 4 * e + 8, "flops": 12.0 * live * e}
    m, n = case["m"], case["n"]
    if kind == "epilogue":
        read = 1 if case["act"] == "none" else 2
        return {"bytes": (read + 1) * m * n * SIZE[case["type"]] + 4 * n,
                "flops": m * n * {"none": 1.0, "relu": 2.0, "gelu": 20.0, "silu": 12.0}[case["act"]]}
    if kind == "norm":
        return {"bytes": m * n * (SIZE[case["x"]] + SIZE[case["y"]]) + 8 * n + 8 * m, "flops": 8.0 * m * n}
    return {"bytes": m * n * (SIZE[case["x"]] * (2 + case["residual"]) + SIZE[case["y"]]) + 12 * n + 8 * m,
            "flops": 14.0 * m * n}


# ---- the operators by their definition, in 64 bits ---------------------------------------------


def exact(case, seed):
    # Nearly all of it is matrix products in 64 bits, at some 20e12 operations a second.
    if work(case)["flops"] > 1.5e11:
        return None
    state = _inputs(case, seed)
    return {"product": _exact_product, "epilogue": _exact_epilogue, "norm": _exact_norm, "norm_grad": _exact_norm_grad,
            "balance": _exact_balance}[case["kind"]](case, state)


def _logistic(z):
    """1 / (1 + exp(-z)) without overflow."""
    small = torch.exp(-z.abs())
    return torch.where(z >= 0, 1.0 / (1.0 + small), small / (1.0 + small))


def _exact_product(case, state):
    m, n, k = case["m"], case["n"], case["k"]
    a, b = state["A"].double(), state["B"].double()
    a = a[:, :k] if case["a"] == "row" else a[:, :m].t()
    b = b[:, :n].t() if case["b"] == "row" else b[:, :k]
    z = (b @ a.t()).t()
    if case["bias"]:
        z = z + state["bias"].double()
    # gelu's tanh form is z times a logistic of twice tanh's argument
    d = {"none": lambda: z, "relu": lambda: z.clamp_min(0.0), "silu": lambda: z * _logistic(z),
         "gelu": lambda: z * _logistic(2.0 * GELU_C * z * (1.0 + GELU_A * z.square()))}[case["act"]]()
    out = {"D": d + state["C"][:, :n].double() if case["residual"] else d}
    if case["z"]:
        out["Z"] = z
    return out


def _exact_epilogue(case, state):
    n = case["n"]
    dy, z = state["dY"][:, :n].double(), state["Z"][:, :n].double()
    if case["act"] == "relu":
        dz = dy * (z > 0)
    elif case["act"] == "none":
        dz = dy
    else:
        # y = z * logistic(v(z)): y' = logistic + z * logistic * (1 - logistic) * v'
        gelu = case["act"] == "gelu"
        s = _logistic(2.0 * GELU_C * z * (1.0 + GELU_A * z.square()) if gelu else z)
        slope = 2.0 * GELU_C * (1.0 + 3.0 * GELU_A * z.square()) if gelu else 1.0
        dz = dy * s * (1.0 + z * (1.0 - s) * slope)
    return {"dZ": dz, "dbias": dz.sum(0)}


def _exact_norm(case, state):
    x = state["X"][:, :case["n"]].double()
    var, mean = torch.var_mean(x, dim=1, correction=0)
    rstd = torch.rsqrt(var + EPS)
    y = torch.addcmul(state["beta"].double(), (x - mean[:, None]) * rstd[:, None], state["gamma"].double())
    return {"Y": y, "mean": mean, "rstd": rstd}


def _exact_norm_grad(case, state):
    # dx_i = sum_j J_ij g_j with J = rstd (I - 1 1'/n - xhat xhat'/n), row by row
    n = case["n"]
    dy = state["dY"][:, :n].double()
    rstd = state["rstd"].double()[:, None]
    xhat = (state["X"][:, :n].double() - state["mean"].double()[:, None]) * rstd
    g = dy * state["gamma"].double()
    along = torch.einsum("ij,ij->i", g, xhat)[:, None] / n
    dx = rstd * (g - g.sum(1, keepdim=True) / n - along * xhat)
    if case["residual"]:
        dx = dx + state["dR"][:, :n].double()
    return {"dX": dx, "dgamma": torch.einsum("ij,ij->j", dy, xhat), "dbeta": dy.sum(0)}


def _exact_balance(case, state):
    # on the CPU; the gradient by differentiating the loss itself
    e = case["experts"]
    ids = state["ids"].cpu()
    members = torch.stack([(ids == i).sum() for i in range(e)])
    live = ((ids >= 0) & (ids < e)).any(1)
    x = state["logits"][:, :e].cpu().double().requires_grad_(True)
    p = torch.softmax(x, 1) if case["scoring"] == "softmax" else _normalised(x)
    mean_score = p[live].mean(0)
    loss = 0.01 * e * torch.dot(members.double() / members.sum(), mean_score)
    gradient, = torch.autograd.grad(loss * state["upstream"].cpu().double()[0], x)
    return {"counts": members.int(), "loss": loss.detach().reshape(1), "dlogits": gradient}


def _normalised(x):
    s = torch.sigmoid(x)
    return s / s.sum(1, keepdim=True)
