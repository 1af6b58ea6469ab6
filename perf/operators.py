"""Measured cases of the embedding, gradient-clipping and row-gradient AdamW operators.

``run`` makes one pass through one operator: in plain torch operations, or
(``own``) through the framework's entry points. Sizes come from the benchmark's
configurations (2B decoder: hidden 2048, kv 256, MLP 8192, embedding
151936 x 2048; VLA stack: hidden 2560 and 1024, MLP 4096; 8 sequences of 2048
tokens) or are generic odd ones.
"""

import math

import torch

own = False

_DT = {"bfloat16": torch.bfloat16, "float32": torch.float32}
_ES = {"bfloat16": 2, "float32": 4}
_BETA1, _BETA2, _EPS = 0.9, 0.95, 1e-8


def listed():
    lookup = {"op": "lookup", "rows": 151936, "dim": 2048, "weight": "bfloat16", "out": "bfloat16", "scale": 1.0,
              "ids": "int64"}
    grad = {"op": "grad", "rows": 151936, "dim": 2048, "grad": "bfloat16", "out": "bfloat16", "scale": 1.0,
            "form": "rows", "pad": -1, "ids": "int64"}
    clip = {"op": "clip", "layers": 4, "hidden": 2048, "kv": 256, "mlp": 8192, "grad": "bfloat16", "out": "bfloat16",
            "norm": 2.0, "max_norm": 1.0}
    adam = {"op": "adamw", "rows": 151936, "dim": 2048, "tokens": 16384, "param": "bfloat16", "grad": "bfloat16",
            "decay": 0.0}
    return [
        # eight sequences generating one token each: the latency of a call
        {**lookup, "name": "lookup-8-tokens", "tokens": 8},
        # the 2B decoder's training batch of 8 x 2048 tokens
        {**lookup, "name": "lookup-2b-batch", "tokens": 16384},
        # fp32 master rows scaled by sqrt(dim), written in bf16; odd sizes
        {**lookup, "name": "lookup-fp32-odd", "tokens": 40961, "rows": 32003, "dim": 1001, "weight": "float32",
         "scale": math.sqrt(1001.0), "ids": "int32"},
        # a short fine-tuning batch in fp32
        {**grad, "name": "grad-rows-512", "tokens": 512, "rows": 32003, "dim": 1024, "grad": "float32",
         "out": "float32", "scale": 32.0},
        # the 2B decoder's batch, as rows and as the dense gradient
        {**grad, "name": "grad-rows-2b-batch", "tokens": 16384},
        {**grad, "name": "grad-dense-2b-batch", "tokens": 16384, "form": "dense"},
        # eight accumulated batches at once, hidden 2560, an eighth of the tokens padding
        {**grad, "name": "grad-rows-131072", "tokens": 131072, "dim": 2560, "scale": 2.0, "pad": 7},
        # a small model's gradients: many small tensors, the latency of a call
        {**clip, "name": "clip-small", "hidden": 72, "kv": 24, "mlp": 200, "max_norm": 0.25},
        # four layers of the 2B decoder in bf16
        {**clip, "name": "clip-2b-4-layers"},
        # the action expert's fp32 accumulators clipped into bf16 gradients
        {**clip, "name": "clip-fp32-expert", "layers": 18, "hidden": 1024, "kv": 1024, "mlp": 4096, "grad": "float32"},
        # the 2B decoder's embedding
        {**adam, "name": "adamw-2b-embedding"},
        # an fp32 embedding of odd sizes with weight decay
        {**adam, "name": "adamw-fp32-odd", "rows": 32003, "dim": 257, "tokens": 3001, "param": "float32",
         "grad": "float32", "decay": 0.01},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["lookup", "grad", "clip", "adamw"])
    types = ["bfloat16", "float32"]
    if op == "clip":
        return {"op": op, "layers": _spread(rng, 1, 20), "hidden": _spread(rng, 17, 1024), "kv": _spread(rng, 8, 512),
                "mlp": _spread(rng, 32, 4096), "grad": rng.choice(types), "out": rng.choice(types),
                "norm": rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]), "max_norm": rng.choice([1.0, 0.3, 1e6])}
    case = {"op": op, "rows": _spread(rng, 100, 151936), "dim": _spread(rng, 16, 2560)}
    if rng.random() < 0.5:
        case["dim"] = max(16, case["dim"] // 64 * 64)
    if op == "adamw":
        param = rng.choice(types)
        return {**case, "dim": min(case["dim"], 2048), "tokens": _spread(rng, 1, 32768), "param": param,
                "grad": param, "decay": 0.0 if param == "bfloat16" else rng.choice([0.0, 0.01])}
    case |= {"scale": rng.choice([1.0, 0.5, math.sqrt(case["dim"])]), "ids": rng.choice(["int64", "int32"])}
    if op == "lookup":
        return {**case, "tokens": _spread(rng, 1, 65536), "weight": rng.choice(types), "out": rng.choice(types)}
    kind = rng.choice(types)
    return {**case, "tokens": _spread(rng, 1, 100000), "grad": kind, "out": rng.choice([kind, "float32"]),
            "form": rng.choice(["rows", "dense"]), "pad": rng.choice([-1, case["rows"] // 2])}


def _tokens(case, gen):
    """Token ids with frequencies falling as 1 / rank, as in text, the ranks spread over the vocabulary."""
    u = torch.rand(case["tokens"], device="cuda", generator=gen, dtype=torch.float64)
    rank = torch.pow(float(case["rows"] + 1), u).long().clamp_(1, case["rows"])
    ids = (rank - 1) * 1000003 % case["rows"]
    if case.get("pad", -1) >= 0:  # the last eighth of every sequence of 2048
        at = torch.arange(ids.numel(), device="cuda") % 2048
        ids = torch.where(at >= 1792, case["pad"], ids)
    return ids


def _distinct(case):
    """Expected number of distinct ids among the case's tokens."""
    r = torch.arange(1, case["rows"] + 1, dtype=torch.float64)
    p = torch.log1p(1.0 / r) / math.log(case["rows"] + 1)
    return float(-torch.expm1(case["tokens"] * torch.log1p(-p)).sum())


def _clip_shapes(case):
    h, kv, mlp = case["hidden"], case["kv"], case["mlp"]
    return [(h, h), (kv, h), (kv, h), (h, h), (mlp, h), (mlp, h), (h, mlp), (h,), (h,)] * case["layers"] + [(h,)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std, dtype="float32"):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).mul_(std).to(_DT[dtype])

    op = case["op"]
    state = {"case": case}
    if op == "lookup":
        state["weight"] = normal(case["rows"], case["dim"], std=0.02, dtype=case["weight"])
        state["ids"] = _tokens(case, gen).to(getattr(torch, case["ids"]))
    elif op == "grad":
        state["ids"] = _tokens(case, gen).to(getattr(torch, case["ids"]))
        state["grad"] = normal(case["tokens"], case["dim"], std=1e-3, dtype=case["grad"])
    elif op == "clip":
        state["grads"] = [normal(*s, std=1e-3, dtype=case["grad"]) for s in _clip_shapes(case)]
        # the results are views of one flat buffer, as data-parallel gradient buckets keep them
        shapes = _clip_shapes(case)
        begins, total = [], 0
        for shape in shapes:
            begins.append(total)
            total += (math.prod(shape) + 63) // 64 * 64
        state["flat"] = torch.zeros(total, device="cuda", dtype=_DT[case["out"]])
        state["out"] = [state["flat"][b:b + math.prod(s)].view(s) for b, s in zip(begins, shapes)]
    else:
        seen = torch.unique(_tokens(case, gen))
        cap = min(case["tokens"], case["rows"])
        state["ids"] = torch.zeros(cap, dtype=torch.int64, device="cuda")
        state["ids"][:seen.numel()] = seen
        state["values"] = normal(cap, case["dim"], std=1e-3, dtype=case["grad"])
        state["values"][seen.numel():] = 0
        state["count"] = torch.full((1,), seen.numel(), dtype=torch.int64, device="cuda")
        state["param"] = normal(case["rows"], case["dim"], std=0.02, dtype=case["param"])
        state["exp_avg"] = normal(case["rows"], case["dim"], std=1e-4)
        state["exp_avg_sq"] = normal(case["rows"], case["dim"], std=1e-3).square_().add_(1e-8)
    return state


_LR, _STEP = 1e-3, 100


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"lookup": _plain_lookup, "grad": _plain_grad, "clip": _plain_clip, "adamw": _plain_adamw}[case["op"]](
        case, state)


def _run_own(case, s):
    from opendm_b200 import embedding as E
    from opendm_b200 import optimizer as O

    if case["op"] == "lookup":
        return E.embedding(s["ids"], s["weight"], scale=case["scale"], out_dtype=_DT[case["out"]])
    if case["op"] == "grad":
        pad = case["pad"] if case["pad"] >= 0 else None
        fn = E.embedding_grad if case["form"] == "dense" else E.embedding_row_grad
        g = fn(s["grad"], s["ids"], case["rows"], scale=case["scale"], padding_idx=pad, dtype=_DT[case["out"]])
        return g if case["form"] == "dense" else {"ids": g.ids, "values": g.values, "count": g.count}
    if case["op"] == "clip":
        total = O.clip_grads(s["grads"], case["max_norm"], norm_type=case["norm"], out=s["out"])
        return {"total": total, "grads": s["flat"]}
    rows = E.RowGrad(case["rows"], s["ids"], s["values"], s["count"])
    O.adamw([s["param"]], [rows], [s["exp_avg"]], [s["exp_avg_sq"]], [_STEP], lr=_LR, beta1=_BETA1, beta2=_BETA2,
            eps=_EPS, weight_decay=case["decay"])
    return {"param": s["param"], "exp_avg": s["exp_avg"], "exp_avg_sq": s["exp_avg_sq"]}


def _plain_lookup(case, s):
    return (s["weight"][s["ids"]].float() * case["scale"]).to(_DT[case["out"]])


def _plain_grad(case, s):
    ids, n, rows, dim = s["ids"].long(), case["tokens"], case["rows"], case["dim"]
    # fp32 results keep what long fp32 sums would lose
    acc = torch.float64 if case["out"] == "float32" else torch.float32
    grad = s["grad"].to(acc)
    if case["pad"] >= 0:
        grad = grad * (ids != case["pad"])[:, None]
    if case["form"] == "dense":
        total = torch.zeros(rows, dim, dtype=acc, device="cuda").index_add_(0, ids, grad)
        return (total * case["scale"]).to(_DT[case["out"]])
    cap = min(n, rows)
    key = torch.where(ids == case["pad"], rows, ids)
    key, order = torch.sort(key, stable=True)
    head = torch.ones_like(key, dtype=torch.bool)
    head[1:] = key[1:] != key[:-1]
    slot = torch.cumsum(head, 0) - 1
    count = (head & (key < rows)).sum().reshape(1)
    # one row more than the result, for the dropped padding's zeros
    total = torch.zeros(cap + 1, dim, dtype=acc, device="cuda").index_add_(0, slot, grad[order])
    out_ids = torch.zeros(cap + 1, dtype=torch.int64, device="cuda").index_copy_(
        0, slot, torch.where(key < rows, key, 0))
    return {"ids": out_ids[:cap], "values": (total[:cap] * case["scale"]).to(_DT[case["out"]]), "count": count}


def _plain_clip(case, s):
    grads = [g.float() for g in s["grads"]]
    p = case["norm"]
    if p == math.inf:
        total = torch.stack([g.abs().max() for g in grads]).max()
    else:
        total = torch.stack([(g.abs() if p == 1.0 else g * g).sum() for g in grads]).sum()
        total = total if p == 1.0 else total.sqrt()
    coef = torch.clamp(case["max_norm"] / (total + 1e-6), max=1.0)
    for g, o in zip(grads, s["out"]):
        o.copy_(g * coef)
    return {"total": total, "grads": s["flat"]}


def _plain_adamw(case, s):
    g = torch.zeros(case["rows"], case["dim"], device="cuda").index_add_(0, s["ids"], s["values"].float())
    m, v, p = s["exp_avg"], s["exp_avg_sq"], s["param"]
    m.mul_(_BETA1).add_(g * (1 - _BETA1))
    v.mul_(_BETA2).add_(g * g * (1 - _BETA2))
    denom = v.sqrt() / math.sqrt(1 - _BETA2 ** _STEP) + _EPS
    p.copy_(p.float() * (1 - _LR * case["decay"]) - (_LR / (1 - _BETA1 ** _STEP)) * (m / denom))
    return {"param": p, "exp_avg": m, "exp_avg_sq": v}


def work(case):
    n = case.get("tokens", 0)
    if case["op"] == "clip":
        elements = sum(math.prod(s) for s in _clip_shapes(case))
        return {"bytes": elements * (_ES[case["grad"]] + _ES[case["out"]]), "flops": 3 * elements}
    rows, dim = case["rows"], case["dim"]
    seen = _distinct(case)
    if case["op"] == "lookup":
        id_bytes = 8 if case["ids"] == "int64" else 4
        return {"bytes": seen * dim * _ES[case["weight"]] + n * dim * _ES[case["out"]] + n * id_bytes,
                "flops": n * dim}
    if case["op"] == "grad":
        id_bytes = 8 if case["ids"] == "int64" else 4
        kept = n if case["pad"] < 0 else n - n // 8
        written = rows * dim if case["form"] == "dense" else min(n, rows) * (dim + 8 / _ES[case["out"]])
        return {"bytes": kept * dim * _ES[case["grad"]] + written * _ES[case["out"]] + n * id_bytes,
                "flops": kept * dim}
    per = 2 * _ES[case["param"]] + 16
    return {"bytes": rows * dim * per + seen * (dim * _ES[case["grad"]] + 8), "flops": 15 * rows * dim}


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "lookup":
        return torch.index_select(s["weight"].to(f64), 0, s["ids"].reshape(-1).long()).mul_(case["scale"])
    if case["op"] == "grad":
        ids = s["ids"].long()
        use = ids != case["pad"]
        kept, grad = ids[use], s["grad"][use].to(f64).mul_(case["scale"])
        if case["form"] == "dense":
            return torch.zeros(case["rows"], case["dim"], dtype=f64, device="cuda").index_add_(0, kept, grad)
        seen, back = torch.unique(kept, return_inverse=True)
        values = torch.zeros(min(case["tokens"], case["rows"]), case["dim"], dtype=f64, device="cuda")
        return {"ids": None, "values": values.index_add_(0, back, grad), "count": None}
    if case["op"] == "clip":
        grads = [g.to(f64) for g in s["grads"]]
        total = torch.linalg.vector_norm(
            torch.stack([torch.linalg.vector_norm(g, case["norm"]) for g in grads]), case["norm"])
        factor = torch.minimum(case["max_norm"] / (total + 1e-6), torch.ones_like(total))
        flat = torch.cat([torch.nn.functional.pad(g.reshape(-1), (0, -g.numel() % 64)) for g in grads])
        return {"total": total, "grads": flat.mul_(factor)}
    p, m, v = (s[k].to(f64) for k in ("param", "exp_avg", "exp_avg_sq"))
    count = int(s["count"])
    g = torch.zeros_like(p)
    g[s["ids"][:count]] = s["values"][:count].to(f64)
    m = _BETA1 * m + (1 - _BETA1) * g
    v = _BETA2 * v + (1 - _BETA2) * g * g
    m_hat = m / (1 - _BETA1 ** _STEP)
    v_hat = v / (1 - _BETA2 ** _STEP)
    p = p - _LR * case["decay"] * p - _LR * m_hat / (v_hat.sqrt() + _EPS)
    return {"param": p, "exp_avg": m, "exp_avg_sq": v}
