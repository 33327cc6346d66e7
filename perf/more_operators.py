"""Low-rank adapters of many requests beside one shared projection, their training step, and the clipping of their
gradients, as a user runs them, with their plain forms.

A bank holds L adapters of rank R for a projection from K to N features: A [L, R, K], B [L, R, N], scaling s [L].
Token t uses adapter i(t) or none:

    y_t = base_t + s_i B_i^T (A_i x_t)            (y_t = base_t without an adapter)

* ``serve``: that product, for single tokens of many requests and for prompts;
* ``train``: the same and, for the gradient dy of y, the gradients of x, of all A and of all B;
* ``clip``: g * min(1, max_norm / (|g| + 1e-6)) for many tensors, with |g| the norm of all their values together.
"""

import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

#: what a serve or train case has when it does not say otherwise
DEFAULTS = {"S": 1, "ragged": False, "none": False}


def _full(case):
    return {**DEFAULTS, **case}


def listed():
    return [
        # one request, one new token, an attention projection: the smallest call of a decode loop
        {"name": "decode one", "op": "serve", "B": 1, "L": 8, "R": 16, "K": 4096, "N": 4096, "type": "bf16"},
        # a decode batch of many tenants, some of them on the bare base model, the widest projection
        {"name": "decode batch", "op": "serve", "B": 64, "L": 32, "R": 16, "K": 4096, "N": 14336, "type": "bf16", "none": True},
        # larger adapters, one for each of 128 requests, the projection back
        {"name": "decode wide", "op": "serve", "B": 128, "L": 128, "R": 64, "K": 14336, "N": 4096, "type": "fp16"},
        # one prompt of one request
        {"name": "prompt one", "op": "serve", "B": 1, "S": 2048, "L": 4, "R": 16, "K": 4096, "N": 4096, "type": "bf16"},
        # right-padded prompts of unequal lengths and different adapters, the widest projection
        {"name": "prompts ragged", "op": "serve", "B": 8, "S": 2048, "L": 8, "R": 64, "K": 4096, "N": 14336, "type": "bf16",
         "ragged": True},
        # tokens of a continuous batch in any order, odd sizes
        {"name": "tokens mixed", "op": "serve", "B": 777, "L": 5, "R": 8, "K": 1032, "N": 2056, "type": "fp16", "none": True},
        # a training batch of several adapters at once
        {"name": "train batch", "op": "train", "B": 4, "S": 1024, "L": 4, "R": 16, "K": 4096, "N": 4096, "type": "bf16"},
        # the largest step: long sequences, large adapters, the widest projection
        {"name": "train long", "op": "train", "B": 4, "S": 4096, "L": 2, "R": 64, "K": 4096, "N": 14336, "type": "bf16"},
        # an odd small step: a rank that is no power of two, padding, sequences without an adapter
        {"name": "train odd", "op": "train", "B": 9, "S": 133, "L": 3, "R": 24, "K": 520, "N": 1288, "type": "fp16",
         "ragged": True, "none": True},
        # the gradients of a layer's adapter, three odd tensors: latency counts
        {"name": "clip small", "op": "clip", "tensors": 3, "size": 5001, "type": "fp32"},
        # the gradients of all adapters of a model, rank 16 on seven projections of 32 layers, as single tensors
        {"name": "clip adapters", "op": "clip", "tensors": 448, "size": 110000, "type": "bf16"},
        # the gradients of one whole layer
        {"name": "clip layer", "op": "clip", "tensors": 9, "size": 24000000, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5, w["flops"] / 400.0)


def _dense(case):
    """Products of the plain form, which takes every token through every adapter."""
    c = _full(case)
    return c["B"] * c["S"] * c["L"] * c["R"] * (c["K"] + c["N"])


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("serve", "train", "clip")}
    dense = {op: max(_dense(c) for c in listed() if c["op"] == op) for op in ("serve", "train")}
    while True:
        op = rng.choice(["serve", "serve", "train", "clip"])
        if op == "clip":
            c = {"op": op, "tensors": _log(rng, 1, 500), "size": _log(rng, 1, 24000000),
                 "type": rng.choice(["bf16", "fp16", "fp32"])}
        else:
            c = {"op": op, "B": _log(rng, 1, 1024) if op == "serve" else _log(rng, 1, 64), "L": _log(rng, 1, 128),
                 "R": rng.choice([1, 4, 8, 16, 16, 24, 32, 64, 128]), "K": 8 * _log(rng, 8, 1792),
                 "N": 8 * _log(rng, 8, 1792), "type": rng.choice(["bf16", "fp16"]), "ragged": rng.random() < 0.5,
                 "none": rng.random() < 0.3}
            c["S"] = 1 if op == "serve" and rng.random() < 0.5 else _log(rng, 2, 4096)
            c["ragged"] = c["ragged"] and c["S"] > 1
        if _cost(c) <= most[op] and (op == "clip" or _dense(c) <= dense[op]):
            return c


def _sizes(c):
    """Numbers of values of the tensors: spread from half of "size" to all of it, odd ones among them."""
    n, s = c["tensors"], c["size"]
    return [max(1, s - (s * i) // (2 * n)) for i in range(n)]


def _lengths(c):
    """Tokens of each request: all the same, or spread from S down to an eighth of it."""
    if not c["ragged"]:
        return [c["S"]] * c["B"]
    return [max(1, c["S"] - (c["S"] * 7 * b) // (8 * max(1, c["B"] - 1))) for b in range(c["B"])]


def _owners(c):
    """Adapters that the requests use: all in turn; with "none" every fourth request uses none (-1)."""
    return [-1 if c["none"] and b % 4 == 3 else b % c["L"] for b in range(c["B"])]


def work(case):
    if case["op"] == "clip":
        n = sum(_sizes(case))
        size = 4 if case["type"] == "fp32" else 2
        return {"bytes": 2 * n * size, "flops": 3 * n}
    c = _full(case)
    B, S, L, R, K, N = (c[k] for k in ("B", "S", "L", "R", "K", "N"))
    users = _owners(c)
    used = len(set(users) - {-1})
    live = sum(n for n, i in zip(_lengths(c), users) if i >= 0)
    weights = 2 * used * R * (K + N)
    if c["op"] == "serve":
        return {"bytes": 2 * (live * K + 2 * B * S * N) + weights, "flops": 2 * live * R * (K + N)}
    # x, dy and base in, y, dx and the gradients of all adapters out
    return {"bytes": 2 * (live * (K + N) + 2 * B * S * N + B * S * K) + weights + 2 * L * R * (K + N),
            "flops": 6 * live * R * (K + N)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = TYPES[case["type"]]

    def rand(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    if case["op"] == "clip":
        # gradients whose norm is some times over the limit: every value is scaled
        return {"grads": [rand(n, scale=0.01) for n in _sizes(case)]}
    c = _full(case)
    B, S, L, R, K, N = (c[k] for k in ("B", "S", "L", "R", "K", "N"))
    users = _owners(c)
    random.Random(seed).shuffle(users)
    x = {"x": rand(B, S, K), "base": rand(B, S, N), "A": rand(L, R, K, scale=K ** -0.5), "B": rand(L, R, N, scale=0.05),
         "s": torch.randint(1, 5, (L,), generator=g, device="cuda").float() / 2,
         "ids": torch.tensor(users, dtype=torch.int32, device="cuda"),
         "counts": torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c["ragged"] else None}
    x["x"][..., :: max(8, K // 8)] *= 10  # a few features are large, as in real activations
    if c["op"] == "train":
        x["dy"] = rand(B, S, N, scale=0.02)
    return x


def prepare(case, seed):
    state = {"case": _full(case), **_inputs(case, seed)}
    if case["op"] == "clip":
        # the optimizer's flat buffer, and each tensor's part of it
        sizes = _sizes(case)
        state["flat"] = torch.empty(sum(sizes), dtype=TYPES[case["type"]], device="cuda")
        state["out"] = list(state["flat"].split(sizes))
        if own:
            import llm_quant_b200 as lq
            state["clipper"] = lq.GradClipper(state["grads"], out=state["out"])
        return state
    if own:
        # kept for as long as the adapters are served, and for all projections of a step
        import llm_quant_b200 as lq
        c = state["case"]
        bank = lq.AdapterBank(c["K"], c["N"], c["L"], c["R"], dtype=TYPES[c["type"]], device="cuda")
        with torch.no_grad():
            bank.lora_A.copy_(state["A"])
            bank.lora_B.copy_(state["B"])
            bank.scaling.copy_(state["s"])
        bank.requires_grad_(c["op"] == "train")
        state["bank"] = bank
        state["batch"] = lq.AdapterBatch(state["ids"], c["L"], c["S"], state["counts"])
    if case["op"] == "train":
        state["x"].requires_grad_(True)
    return state


# ---- the operators ---------------------------------------------------------------------------------------------------------

def _chosen(c, ids, counts, s):
    """[B * S, L * R]: the scaling where a token uses an adapter, 0 where it does not."""
    m = (ids[:, None] == torch.arange(c["L"], device="cuda")).float() * s
    m = m[:, None, :].expand(-1, c["S"], -1)
    if counts is not None:
        m = m * (torch.arange(c["S"], device="cuda") < counts[:, None])[..., None]
    return m.reshape(-1, c["L"], 1).expand(-1, -1, c["R"]).reshape(-1, c["L"] * c["R"])


def _plain(c, x, base, A, B, s, ids, counts, dy):
    dt = x.dtype
    m = _chosen(c, ids, counts, s)
    A, B = A.float().flatten(0, 1), B.float().flatten(0, 1)
    x2 = x.float().flatten(0, 1)
    u = (x2 @ A.T) * m
    y = (base.float() + (u @ B).view(base.shape)).to(dt)
    if dy is None:
        return y
    d2 = dy.float().flatten(0, 1)
    v = (d2 @ B.T) * m
    return [y, (v @ A).view(x.shape).to(dt), (v.T @ x2).view(c["L"], c["R"], -1).to(dt),
            (u.T @ d2).view(c["L"], c["R"], -1).to(dt)]


def run(state):
    c = state["case"]
    if c["op"] == "clip":
        if own:
            norm = state["clipper"].clip(1.0)
        else:
            norm = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt()
            coef = (1.0 / (norm + 1e-6)).clamp(max=1.0)
            torch.cat([(g.double() * coef).to(g.dtype) for g in state["grads"]], out=state["flat"])
            norm = norm.float()
        return [norm, state["flat"]]
    if not own:
        with torch.no_grad():
            return _plain(c, *(state[k] for k in ("x", "base", "A", "B", "s", "ids", "counts")), state.get("dy"))
    bank = state["bank"]
    y = bank(state["x"], state["batch"], state["base"])
    if c["op"] == "serve":
        return y
    return [y.detach(), *torch.autograd.grad(y, (state["x"], bank.lora_A, bank.lora_B), state["dy"])]


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def exact(case, seed):
    i = _inputs(case, seed)
    if case["op"] == "clip":
        total = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in i["grads"]))
        factor = min(1.0, 1.0 / (total + 1e-6))
        return [torch.tensor(total, dtype=torch.float64), torch.cat([g.to(torch.float64) * factor for g in i["grads"]])]
    c = _full(case)
    train = c["op"] == "train"
    y = i["base"].double()
    dx = torch.zeros(i["x"].shape, dtype=torch.float64, device="cuda") if train else None
    dA, dB = (torch.zeros(i[k].shape, dtype=torch.float64, device="cuda") if train else None for k in "AB")
    scale = i["s"].tolist()
    for b, (owner, n) in enumerate(zip(i["ids"].tolist(), _lengths(c))):
        if owner < 0:
            continue
        x, A, B = i["x"][b, :n].double(), i["A"][owner].double(), i["B"][owner].double()
        low = torch.einsum("tk,rk->tr", x, A) * scale[owner]
        y[b, :n] += torch.einsum("tr,rn->tn", low, B)
        if train:
            d = i["dy"][b, :n].double()
            back = torch.einsum("tn,rn->tr", d, B) * scale[owner]
            dx[b, :n] = torch.einsum("tr,rk->tk", back, A)
            dA[owner] += torch.einsum("tr,tk->rk", back, x)
            dB[owner] += torch.einsum("tr,tn->rn", low, d)
    return [y, dx, dA, dB] if train else y
