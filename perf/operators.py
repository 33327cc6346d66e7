"""The operators of the 4-bit KV cache (llm_quant_b200.PackedKVCache) as a user runs them, with their plain forms.

A cache holds K and V of one layer in 4 bits a value: for each token and kv head, over the head dim,

    lo = min(0, min x)   hi = max(0, max x)   scale = bf16((hi - lo) / 15)
    zero = clamp(rint(-lo / scale), 0, 15)    code = clamp(rint(x / scale) + zero, 0, 15)
    value = (code - zero) * scale             (scale 0: zero = code = 0)

Four operators work on it:

* ``write``: a chunk is quantized into the cache and read out as values;
* ``attend``: softmax attention of new queries over the cached tokens, for single tokens and for chunks of a
  prompt, with a tanh cap, a distance bias, a sliding window and a prefix that every query sees;
* ``weigh``: the same, and each cached token collects the attention weight that it got;
* ``evict``: a chunk is appended, then every sequence is cut back to the tokens with the greatest collected weight.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}

#: what a case has when it does not say otherwise
DEFAULTS = {"ragged": False, "causal": False, "softcap": 0.0, "bias": False, "window": 0, "prefix": 0,
            "keep": 0, "recent": 0, "sinks": 0, "G": 1, "S": 1}


def _full(case):
    return {**DEFAULTS, **case}


def listed():
    return [
        # a batch of prompts of unequal lengths, right-padded, written after a reset and read out
        {"name": "write prompt", "op": "write", "B": 8, "H": 8, "D": 128, "S": 2048, "type": "bf16", "ragged": True},
        # a short odd chunk of one sequence: latency counts
        {"name": "write short", "op": "write", "B": 1, "H": 4, "D": 64, "S": 37, "type": "fp16"},
        # one sequence, one new token: the smallest call of a decode loop
        {"name": "decode single", "op": "attend", "B": 1, "H": 8, "G": 4, "D": 128, "T": 500, "type": "bf16"},
        # the sizes of this repository's decode-attention benchmark
        {"name": "decode batch", "op": "attend", "B": 8, "H": 8, "G": 4, "D": 128, "T": 8192, "type": "fp16"},
        # a serving batch of unequal lengths with long sequences
        {"name": "decode long ragged", "op": "attend", "B": 16, "H": 8, "G": 8, "D": 128, "T": 20011, "type": "bf16",
         "ragged": True},
        # a chunk of a long prompt against what is cached of it: bound by arithmetic
        {"name": "prompt chunk", "op": "attend", "B": 1, "H": 8, "G": 4, "D": 128, "T": 8192, "S": 2048, "type": "bf16",
         "causal": True},
        # prompts of unequal lengths whose prefix is seen by all their tokens, scores capped, older tokens out of a window
        {"name": "prompt capped window", "op": "attend", "B": 3, "H": 4, "G": 2, "D": 64, "T": 1500, "S": 777,
         "type": "fp16", "ragged": True, "causal": True, "softcap": 30.0, "window": 512, "prefix": 100},
        # decode with capped scores and a bias that falls with the distance, one query head for each kv head
        {"name": "decode capped bias", "op": "attend", "B": 8, "H": 16, "G": 1, "D": 64, "T": 3001, "type": "bf16",
         "ragged": True, "causal": True, "softcap": 50.0, "bias": True},
        # the decode step of a cache that will evict: weights are collected
        {"name": "weigh decode", "op": "weigh", "B": 8, "H": 8, "G": 4, "D": 128, "T": 4096, "type": "bf16",
         "ragged": True},
        # the prompt's own weights, collected while it is processed
        {"name": "weigh prompt", "op": "weigh", "B": 2, "H": 8, "G": 4, "D": 128, "T": 2048, "S": 1024, "type": "bf16",
         "causal": True},
        # a decode loop with a budget: each token pushes another one out
        {"name": "evict one", "op": "evict", "B": 4, "H": 8, "D": 128, "S": 1, "type": "bf16", "keep": 1000,
         "recent": 128, "sinks": 4},
        # prompt chunks through a budget
        {"name": "evict chunk", "op": "evict", "B": 8, "H": 8, "D": 128, "S": 1024, "type": "fp16", "keep": 8192,
         "recent": 2048, "sinks": 4, "ragged": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.5, w["flops"] / 800.0)


def _all_pairs(case):
    c = _full(case)
    return c["B"] * c["H"] * c["G"] * c["S"] * c.get("T", 0)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("write", "attend", "weigh", "evict")}
    pairs = max(_all_pairs(c) for c in listed())
    values = max(c["B"] * c["H"] * c["D"] * c.get("T", 0) for c in listed())
    while True:
        op = rng.choice(["write", "attend", "attend", "attend", "weigh", "evict"])
        c = {"op": op, "B": _log(rng, 1, 16), "H": rng.choice([1, 2, 4, 5, 8, 16]), "D": rng.choice([64, 128]),
             "type": rng.choice(["bf16", "fp16"]), "ragged": rng.random() < 0.5}
        if op == "write":
            c["S"] = _log(rng, 1, 4096)
        elif op == "evict":
            c["keep"] = _log(rng, 64, 8192)
            c["S"] = min(c["keep"], _log(rng, 1, 1024))
            c["sinks"] = rng.choice([0, 4])
            c["recent"] = min(c["keep"] - c["sinks"], _log(rng, 1, 2048))
        else:
            c["G"] = rng.choice([1, 2, 3, 4, 8])
            c["T"] = _log(rng, 16, 20011)
            c["S"] = 1 if rng.random() < 0.5 else min(c["T"], _log(rng, 2, 2048))
            c["causal"] = c["S"] > 1 or rng.random() < 0.5
            if rng.random() < 0.4:
                c["softcap"] = rng.choice([20.0, 30.0, 50.0])
            if rng.random() < 0.3:
                c["bias"] = True
            if rng.random() < 0.3:
                c["window"] = _log(rng, 8, 4096)
            if rng.random() < 0.3:
                c["prefix"] = _log(rng, 1, c["T"])
        if _cost(c) <= most[op] and _all_pairs(c) <= pairs and c["B"] * c["H"] * c["D"] * c.get("T", 0) <= values:
            return c


def _lengths(c, longest):
    """Tokens of each sequence: all the same, or spread from the longest down to an eighth of it."""
    if not c["ragged"] or c["B"] == 1:
        return [longest] * c["B"]
    return [max(1, longest - (longest * 7 * b) // (8 * (c["B"] - 1))) for b in range(c["B"])]


def _counts(c):
    """New tokens of each sequence: the chunk, less where a sequence is shorter."""
    if c["op"] == "write":
        return _lengths(c, c["S"])
    if c["op"] == "evict":
        return [c["S"]] * c["B"]
    return [min(c["S"], t) for t in _lengths(c, c["T"])]


def _visible(c, n, cnt):
    """Pairs of one query head's query and a cached token that it sees, for a sequence of n tokens."""
    pairs = 0
    for i in range(cnt):
        p = n - cnt + i
        last = p if c["causal"] else n - 1
        first = max(0, p - c["window"] + 1) if c["window"] else 0
        pre = min(c["prefix"], n)
        pairs += max(0, last - first + 1) + (min(pre, first) + max(0, pre - 1 - last) if last >= first else pre)
    return pairs


def work(case):
    c = _full(case)
    BH, D = c["B"] * c["H"], c["D"]
    token = 2 * (D // 2 + 4)  # codes, scale and zero of K and of V
    if c["op"] == "write":
        n = sum(_counts(c)) * c["H"]
        return {"bytes": n * (4 * D + token + 8) + BH * c["S"] * 4 * D, "flops": 0}
    if c["op"] == "evict":
        # the chunk in; weights and positions of all slots; the survivors among the new tokens move; the values out
        moved = BH * min(c["S"], c["keep"])
        return {"bytes": moved * (4 * D + 3 * token) + 8 * BH * (c["keep"] + c["S"]) + BH * c["keep"] * (token + 4 * D),
                "flops": 0}
    lens, cnts = _lengths(c, c["T"]), _counts(c)
    cached = 0
    for n, cnt in zip(lens, cnts):
        first = n - cnt - c["window"] + 1 if c["window"] else 0  # the oldest token that any query sees
        cached += n if first <= 0 else n - first + min(c["prefix"], first)
    masked = (c["causal"] and c["S"] > 1) or c["window"] or c["prefix"] or c["bias"]
    per_token = token + (4 if masked else 0) + (8 if c["op"] == "weigh" else 0)
    pairs = sum(_visible(c, n, cnt) for n, cnt in zip(lens, cnts))
    return {"bytes": cached * c["H"] * per_token + 2 * 2 * BH * c["G"] * c["S"] * D,
            "flops": 4 * D * pairs * c["H"] * c["G"]}


# ---- inputs --------------------------------------------------------------------------------------------------------

def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    c = _full(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, H, D, S, dt = c["B"], c["H"], c["D"], c["S"], TYPES[c["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def projected(heads, tokens, factor):
        """[B, heads, tokens, D] as a projection gives it: tokens before heads in memory."""
        return (normal(B, tokens, heads, D) * factor).to(dt).transpose(1, 2)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    channel = 0.5 + 1.5 * torch.rand(D, generator=g, device="cuda") ** 4  # a few channels of K are larger
    x = {"counts": ints(_counts(c)) if c["ragged"] else None}
    if c["op"] == "write":
        return {**x, "k": projected(H, S, channel), "v": projected(H, S, 1.0)}
    if c["op"] == "evict":
        lens = _lengths(c, c["keep"])
        x |= {"k0": projected(H, c["keep"], channel), "v0": projected(H, c["keep"], 1.0),
              "k": projected(H, S, channel), "v": projected(H, S, 1.0)}
        # collected weight is heavy-tailed: few tokens get most of it
        x["mass0"] = torch.exp(1.5 * normal(B, H, c["keep"]) - 3.0)
    else:
        lens = _lengths(c, c["T"])
        x |= {"k0": projected(H, c["T"], channel), "v0": projected(H, c["T"], 1.0),
              "q": projected(H * c["G"], S, 1.3)}
        x["slopes"] = None
        if c["bias"]:  # 2^(-8 i / n) for the n heads, a usual choice
            n = H * c["G"]
            x["slopes"] = torch.exp2(-8.0 * torch.arange(1, n + 1, device="cuda", dtype=torch.float32) / n)
        x["prefix"] = ints([min(c["prefix"], n) for n in lens]) if c["prefix"] else None
    x["lens0"] = ints(lens)
    return x


def prepare(case, seed):
    c = _full(case)
    x = _inputs(case, seed)
    room = {"write": c["S"], "evict": c["keep"] + c["S"]}.get(c["op"]) or c["T"]
    s = {"case": c, **x}
    if own:
        from llm_quant_b200 import PackedKVCache
        s["cache"] = PackedKVCache(1, max_seq_len=room)
        if c["op"] != "write":
            s["cache"].append(0, x["k0"], x["v0"], counts=x["lens0"])
            if c["op"] == "evict":
                live = torch.arange(c["keep"], device="cuda") < x["lens0"][:, None, None]
                s["cache"].attention_mass(0).copy_(torch.where(live, x["mass0"], 0.0))
    else:
        s["cache"] = _new(c, room)
        if c["op"] != "write":
            _append(s["cache"], x["k0"], x["v0"], x["lens0"])
            if c["op"] == "evict":
                live = torch.arange(c["keep"], device="cuda") < x["lens0"][:, None, None]
                s["cache"]["mass"][:, :, :c["keep"]] = torch.where(live, x["mass0"], 0.0)
    for key in ("k0", "v0", "mass0", "lens0"):
        s.pop(key, None)
    return s


# ---- the plain form: elementary operations on a cache that is a dict of tensors ------------------------------------------

def _new(c, room):
    shape = (c["B"], c["H"], room + 1)  # the last slot is spare: what is padding is written there

    def side():
        return {"codes": torch.zeros(*shape, c["D"] // 2, dtype=torch.uint8, device="cuda"),
                "scale": torch.zeros(*shape, 1, dtype=torch.bfloat16, device="cuda"),
                "zero": torch.zeros(*shape, 1, dtype=torch.uint8, device="cuda")}

    return {"k": side(), "v": side(), "pos": torch.full(shape, -1, dtype=torch.int32, device="cuda"),
            "mass": torch.zeros(shape, device="cuda"),
            "len": torch.zeros(c["B"], dtype=torch.int32, device="cuda"),
            "next": torch.zeros(c["B"], dtype=torch.int32, device="cuda")}


def _quantize(x):
    x = x.float()
    lo = x.amin(-1, keepdim=True).clamp(max=0.0)
    hi = x.amax(-1, keepdim=True).clamp(min=0.0)
    scale = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16)  # by a tensor: a number is multiplied by its reciprocal
    s = scale.float()
    safe = torch.where(s == 0, 1.0, s)
    zero = torch.round(-lo / safe).clamp(0, 15)
    code = (torch.round(x / safe) + zero).clamp(0, 15).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale, zero.to(torch.uint8)


def _values(side, n):
    """fp32 values of the first n slots."""
    p = side["codes"][:, :, :n]
    code = torch.stack((p & 15, p >> 4), -1).flatten(-2)
    return (code.float() - side["zero"][:, :, :n].float()) * side["scale"][:, :, :n].float()


def _append(cache, k, v, counts):
    S = k.shape[2]
    cnt = torch.full_like(cache["len"], S) if counts is None else counts
    i = torch.arange(S, device="cuda")
    slot = torch.where(i < cnt[:, None], cache["len"][:, None] + i, cache["pos"].shape[2] - 1)  # [B, S]; padding: spare
    b = torch.arange(k.shape[0], device="cuda")[:, None]
    for side, x in (("k", k), ("v", v)):
        for name, y in zip(("codes", "scale", "zero"), _quantize(x)):
            cache[side][name][b, :, slot] = y.transpose(1, 2)
    cache["pos"][b, :, slot] = (cache["next"][:, None] + i).int()[..., None]
    cache["mass"][b, :, slot] = 0.0
    cache["len"] += cnt
    cache["next"] += cnt


def _read(cache, n, dtype):
    live = (torch.arange(n, device="cuda") < cache["len"][:, None])[:, None, :, None]
    return [torch.where(live, _values(cache[side], n), 0.0).to(dtype) for side in ("k", "v")]


def _attend(c, cache, q, counts, slopes, prefix, weigh):
    B, H, G, S, D, T = c["B"], c["H"], c["G"], c["S"], c["D"], c["T"]
    k, v = _values(cache["k"], T), _values(cache["v"], T)
    x = torch.matmul(q.float().reshape(B, H, G * S, D), k.transpose(-1, -2)).view(B, H, G, S, T) * D ** -0.5
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    i = torch.arange(S, device="cuda", dtype=torch.int32)
    cnt = torch.full_like(cache["len"], S) if counts is None else counts
    at = (cache["next"] - cnt)[:, None] + i  # [B, S]: positions of the queries
    pos = cache["pos"][:, :, None, None, :T]
    back = at[:, None, None, :, None] - pos  # [B, H, 1, S, T]: how far back a token is
    if slopes is not None:
        x = x - slopes.view(H, G, 1, 1) * back.abs().float()
    sees = torch.ones_like(back, dtype=torch.bool)
    if c["causal"]:
        sees &= back >= 0
    if c["window"]:
        sees &= back < c["window"]
    if prefix is not None:
        sees |= pos < prefix[:, None, None, None, None]
    sees &= (torch.arange(T, device="cuda") < cache["len"][:, None])[:, None, None, None, :]
    sees &= (i < cnt[:, None])[:, None, None, :, None]
    x = x.masked_fill_(~sees, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = torch.matmul(p.view(B, H, G * S, T), v).view(B, H * G, S, D).to(q.dtype)
    if not weigh:
        return out
    cache["mass"][:, :, :T] += p.sum((2, 3))
    return [out, cache["mass"][:, :, :T]]


def _evict(cache, keep, recent, sinks):
    n = cache["len"][:, None, None]
    slot = torch.arange(cache["pos"].shape[2], device="cuda")
    safe = (cache["pos"] >= cache["next"][:, None, None] - recent) | (cache["pos"] < sinks)
    key = torch.where(safe, math.inf, cache["mass"])
    key = torch.where(slot < n, key, -1.0)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(safe).scatter_(-1, order[:, :, :keep], True) & (slot < n)
    # the holes below `keep` are filled, in order, by what is kept at or above it
    rank = torch.where(slot < keep, (~kept).cumsum(-1), 0)
    late = torch.where(kept & (slot >= keep), 0, 1).argsort(dim=-1, stable=True)  # kept slots at or above `keep` first
    src = torch.where(kept[:, :, :keep] | (n <= keep), slot[:keep], late.gather(-1, (rank[:, :, :keep] - 1).clamp(min=0)))
    for side in ("k", "v"):
        for y in cache[side].values():
            y[:, :, :keep] = y.gather(2, src[..., None].expand(-1, -1, -1, y.shape[3]))
    for name, empty in (("pos", -1), ("mass", 0.0)):
        cache[name][:, :, :keep] = cache[name].gather(2, src)
        cache[name][:, :, keep:] = empty
    cache["len"].clamp_(max=keep)


def run(state):
    c, cache = state["case"], state["cache"]
    dt = TYPES[c["type"]]
    if c["op"] == "write":
        if own:
            cache.reset(0)
            return list(cache.update(0, state["k"], state["v"], counts=state["counts"], dtype=dt))
        cache["len"].zero_()
        cache["next"].zero_()
        _append(cache, state["k"], state["v"], state["counts"])
        return _read(cache, c["S"], dt)
    if c["op"] == "evict":
        keep = c["keep"]
        if own:
            cache.append(0, state["k"], state["v"])
            cache.evict(0, keep, recent=c["recent"], sinks=c["sinks"])
            return [cache.positions(0), cache.attention_mass(0), cache.lengths(0), *cache.get(0, dtype=dt)]
        _append(cache, state["k"], state["v"], None)
        _evict(cache, keep, c["recent"], c["sinks"])
        return [cache["pos"][:, :, :keep], cache["mass"][:, :, :keep], cache["len"], *_read(cache, keep, dt)]
    weigh = c["op"] == "weigh"
    if own:
        out = cache.attend(0, state["q"], causal=c["causal"], counts=state["counts"], softcap=c["softcap"],
                           slopes=state["slopes"], window=c["window"], prefix=state["prefix"], accumulate=weigh)
        return [out, cache.attention_mass(0)] if weigh else out
    return _attend(c, cache, state["q"], state["counts"], state["slopes"], state["prefix"], weigh)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def _exact_values(x):
    """What the cache holds for x, in 64 bits but for the scale, which is stored in bf16 by definition."""
    x = x.double()
    zeros = torch.zeros_like(x[..., :1])
    lo = torch.cat((x, zeros), -1).min(-1, keepdim=True).values
    hi = torch.cat((x, zeros), -1).max(-1, keepdim=True).values
    s = ((hi - lo) / torch.full_like(hi, 15.0)).to(torch.bfloat16).double()
    t = torch.where(s > 0, s, torch.ones_like(s))
    zero = torch.minimum((-lo / t).round(), torch.full_like(t, 15.0))
    code = ((x / t).round() + zero).clamp(0.0, 15.0)
    return (code - zero) * s


def exact(case, seed):
    c = _full(case)
    x = _inputs(case, seed)
    B, H, G, S, D = c["B"], c["H"], c["G"], c["S"], c["D"]
    if c["op"] == "write":
        out = []
        for name in ("k", "v"):
            y = _exact_values(x[name])
            for b, n in enumerate(_counts(c)):
                y[b, :, n:] = 0.0
            out.append(y)
        return out
    lens = x["lens0"].tolist()
    k, v = _exact_values(x["k0"]), _exact_values(x["v0"])
    if c["op"] == "evict":
        return _exact_evict(c, x, lens, k, v)
    T = c["T"]
    cnts = _counts(c) if c["ragged"] else [S] * B
    out = torch.zeros(B, H * G, S, D, dtype=torch.float64, device="cuda")
    mass = torch.zeros(B, H, T, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, m = lens[b], cnts[b]
        tok = torch.arange(n, device="cuda")
        qp = n - m + torch.arange(m, device="cuda")
        far = qp[:, None] - tok[None, :]
        ok = torch.ones(m, n, dtype=torch.bool, device="cuda")
        if c["causal"]:
            ok &= far >= 0
        if c["window"]:
            ok &= far < c["window"]
        if c["prefix"]:
            ok |= (tok < min(c["prefix"], n))[None, :]
        for h in range(H * G):
            z = x["q"][b, h, :m].double() @ k[b, h // G, :n].T / math.sqrt(D)
            if c["softcap"]:
                z = torch.tanh(z / c["softcap"]) * c["softcap"]
            if c["bias"]:
                z = z - x["slopes"][h].double() * far.abs().double()
            z = torch.where(ok, z, torch.full_like(z, -math.inf))
            w = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
            out[b, h, :m] = w @ v[b, h // G, :n]
            mass[b, h // G, :n] += w.sum(0)
    return [out, mass] if c["op"] == "weigh" else out


def _exact_evict(c, x, lens, k, v):
    B, H, S, D, keep = c["B"], c["H"], c["S"], c["D"], c["keep"]
    kn, vn = _exact_values(x["k"]), _exact_values(x["v"])
    positions = torch.full((B, H, keep), -1, dtype=torch.int32)
    mass = torch.zeros(B, H, keep, dtype=torch.float64)
    K = torch.zeros(B, H, keep, D, dtype=torch.float64, device="cuda")
    V = torch.zeros_like(K)
    m0 = x["mass0"].double().cpu()
    for b in range(B):
        n = lens[b]
        for h in range(H):
            weight = m0[b, h, :n].tolist() + [0.0] * S
            order = list(range(n + S))
            if n + S > keep:
                first = n + S - c["recent"]
                best = sorted(order, key=lambda t: (not (t >= first or t < c["sinks"]), -weight[t], t))
                kept = sorted(best[:keep])
                late = iter([t for t in kept if t >= keep])
                stays = set(kept)
                order = [t if t in stays else next(late) for t in range(keep)]
            m = len(order)
            at = torch.tensor(order)
            positions[b, h, :m] = at.int()
            mass[b, h, :m] = torch.tensor(weight, dtype=torch.float64)[at]
            K[b, h, :m] = torch.cat((k[b, h, :n], kn[b, h]))[at.cuda()]
            V[b, h, :m] = torch.cat((v[b, h, :n], vn[b, h]))[at.cuda()]
    return [positions, mass, torch.tensor([min(n + S, keep) for n in lens], dtype=torch.int32), K, V]
