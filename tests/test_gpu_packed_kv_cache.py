"""GPU numerics: the 4-bit KV cache (PackedKVCache -> lq_kv4_*).

What is written is compared for equality with the quantization's definition in
numpy fp32 (single operations, no contraction).  Attention is compared with
float64 softmax attention over the values that the cache holds.

Tolerance of attention, per output element (p: exact probabilities, v: values,
s_v: V scales, T tokens):
* scores: products are exact, an accumulator takes at most 8 + 1 additions
  (16-wide MMA steps of D = 128 in two chains, then their sum), each off by at
  most 2^-22 of the largest partial sum; partial sums are at most
  a = |scale| sum_d |q_d| 15 s_k (codes are uncentred).  With the factors after
  it: dx <= 12 * 2^-22 * max a.  A cap only shrinks it and adds its own
  2^-21 * cap; a bias adds 2^-23 of itself where p is not negligible.
* p: relative 2 (dx + 2^-20) from numerator and denominator;
* P is rounded to f16 (2^-11) for 16-bit queries, to 22 bits for fp32 ones, and
  below 2^-14 of the largest product by 2^-25 absolute (each is at most 1 in
  units of the largest p s_v): 2^-24 * T * 15 * max s_v covers it;
* accumulation over T / 16 MMA steps of uncentred codes: (T / 16 + 8) 2^-22 *
  sum p 15 s_v;
* the output's own rounding, half a unit in the last place.
The collected weight is the sum of p over the rows: relative 2 (dx + 2^-20),
plus 2^-23 for each of the additions.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ALL = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def L():
    import llm_quant_b200
    return llm_quant_b200


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv(B, H, S, D, dtype, seed, spread=True):
    """[B, H, S, D] views of a projection's [B, S, H, D], some channels larger."""
    g = _gen(seed)
    ch = 0.5 + 1.5 * torch.rand(D, generator=g, device="cuda") ** 4 if spread else 1.0
    k = (torch.randn(B, S, H, D, generator=g, device="cuda") * ch).to(dtype).transpose(1, 2)
    v = torch.randn(B, S, H, D, generator=g, device="cuda").to(dtype).transpose(1, 2)
    return k, v


def _q(B, Hq, S, D, dtype, seed):
    return (torch.randn(B, S, Hq, D, generator=_gen(seed), device="cuda") * 1.3).to(dtype).transpose(1, 2)


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def quantized(x):
    """The definition, in fp32 numpy: (value fp32, scale)."""
    x = x.float().cpu().numpy()
    lo = np.minimum(x.min(-1, keepdims=True), np.float32(0))
    hi = np.maximum(x.max(-1, keepdims=True), np.float32(0))
    s = torch.from_numpy((hi - lo) / np.float32(15)).to(torch.bfloat16).float().numpy()
    s = np.where(s < 2.0 ** -100, np.float32(0), s)
    d = np.where(s == 0, np.float32(1), s)
    with np.errstate(invalid="ignore"):  # tokens that are not finite
        z = np.minimum(np.rint(-lo / d), np.float32(15))
        c = np.clip(np.rint(x / d) + z, np.float32(0), np.float32(15))
        return (c - z) * s, s


def reference(cache, layer, q, scale=None, causal=False, counts=None, softcap=0.0, slopes=None, window=0, prefix=None,
              mass=False):
    """float64 attention over the values held, and the bounds: (out, bound, mass, mass bound, rows that see nothing)."""
    k, v = (x.double() for x in cache.get(layer))
    st = cache._layers[layer]
    n, pos = cache.lengths(layer), cache.positions(layer).long()
    B, H, T, D = k.shape
    Hq, S = q.shape[1], q.shape[2]
    G = Hq // H
    sm = D ** -0.5 if scale is None else scale
    qd = q.double().reshape(B, H, G, S, D)
    x = torch.einsum("bhgsd,bhtd->bhgst", qd, k) * sm
    s_k = st.params[:, :, :T, 0].bitwise_left_shift(16).view(torch.float32).double()
    s_v = st.params[:, :, :T, 1].bitwise_left_shift(16).view(torch.float32).double()
    live = torch.arange(T, device="cuda") < n[:, None]
    s_k, s_v = (torch.where(live[:, None], s, 0.0) for s in (s_k, s_v))
    a = abs(sm) * qd.abs().sum(-1) * 15 * s_k.amax(-1)[:, :, None, None]  # [B, H, G, S]
    dx = 12 * 2.0 ** -22 * a
    if softcap:
        x = softcap * torch.tanh(x / softcap)
        dx = dx + 2.0 ** -21 * softcap
    i = torch.arange(S, device="cuda")
    cnt = torch.full((B,), S, device="cuda") if counts is None else counts.long().clamp(0, S)
    at = (st.state[B:2 * B].long() - cnt)[:, None] + i
    back = at[:, None, None, :, None] - pos[:, :, None, None, :]
    if slopes is not None:
        bias = slopes.double().view(H, G, 1, 1) * back.abs().double()
        x = x - bias
        dx = dx + 2.0 ** -20 * 64  # beyond a bias of 64 the probability is negligible
    sees = torch.ones_like(back, dtype=torch.bool)
    if causal:
        sees = sees & (back >= 0)
    if window:
        sees = sees & (back < window)
    if prefix is not None:
        sees = sees | (pos[:, :, None, None, :] < prefix.long()[:, None, None, None, None])
    sees = sees & live[:, None, None, None] & (i < cnt[:, None])[:, None, None, :, None]
    x = torch.where(sees, x, -math.inf)
    p = torch.softmax(x, -1).nan_to_num(nan=0.0)
    out = torch.einsum("bhgst,bhtd->bhgsd", p, v)
    rel = 2 * (dx + 2.0 ** -20)[..., None]
    rel_p = rel + (2.0 ** -11 if q.dtype != torch.float32 else 2.0 ** -21)
    spread = torch.einsum("bhgst,bhtd->bhgsd", p, v.abs())
    weight = torch.einsum("bhgst,bht->bhgs", p, s_v)[..., None] * 15
    top = s_v.amax(-1)[:, :, None, None, None] * 15
    bound = rel_p * spread + (T / 16 + 8) * 2.0 ** -22 * weight + 2.0 ** -24 * T * top \
        * (1.0 if q.dtype != torch.float32 else 2.0 ** -10) + out.abs() * EPS[q.dtype]
    m = p.sum((2, 3))
    mb = (p * rel).sum((2, 3)) + (G * S + 8) * 2.0 ** -23 * m + 1e-30
    return out.reshape(B, Hq, S, D), bound.reshape(B, Hq, S, D), m, mb, (p.sum(-1) == 0).reshape(B, Hq, S)


def check(L, cache, q, layer=0, **kw):
    ref, bound, m, mb, blind = reference(cache, layer, q, **kw)
    before = cache.attention_mass(layer).double().clone()
    out = cache.attend(layer, q, **kw)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    assert torch.isfinite(out).all()
    err = (out.double() - ref).abs()
    assert (err <= bound).all(), (float((err / bound).max()), float(err.max()))
    assert (out[blind] == 0).all()
    assert torch.equal(cache.attention_mass(layer).double(), before)
    out2 = cache.attend(layer, q, accumulate=True, **kw)
    assert torch.equal(out2, out)
    assert cache._layers[layer].state[-1].item() == 0  # no wait on the device ran out
    got = cache.attention_mass(layer).double() - before
    err = (got - m).abs()
    mb = mb + before.abs() * 2.0 ** -23 + m * 2.0 ** -23
    assert (err <= mb).all(), (float((err / mb).max()), float(err.max()))
    return out


# ---- writing ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ALL)
def test_written_values_are_the_definitions(L, dtype, D):
    cache = L.PackedKVCache(1, 300)
    ks, vs = [], []
    for i, S in enumerate((1, 15, 17, 1, 33, 100, 64, 3)):
        k, v = _kv(2, 3, S, D, dtype, 10 * D + i)
        cache.append(0, k, v)
        ks.append(k), vs.append(v)
    K, V = cache.get(0)
    assert K.shape == (2, 3, 234, D) and cache.seq_len == 234
    for got, parts in ((K, ks), (V, vs)):
        ref, _ = quantized(torch.cat(parts, 2))
        assert np.array_equal(got.cpu().numpy(), ref)
    assert cache.lengths(0).tolist() == [234, 234]
    assert torch.equal(cache.positions(0), torch.arange(234, device="cuda", dtype=torch.int32).expand(2, 3, -1))
    for dt in (torch.float16, torch.bfloat16):
        k16, v16 = cache.get(0, dt)
        assert torch.equal(k16, K.to(dt)) and torch.equal(v16, V.to(dt))


def test_counts_and_padding(L):
    cache = L.PackedKVCache(2, 64)
    parts = [[], [], []]
    for i, cnt in enumerate([(5, 0, 7), (1, 7, 0), (20, 3, 16), (0, 0, 0), (4, 99, -3)]):
        S = max(1, min(max(cnt), 20))
        k, v = _kv(3, 2, S, 64, torch.bfloat16, i)
        for b, n in enumerate(cnt):  # padding is not read
            k[b, :, min(max(n, 0), S):] = float("nan")
            parts[b].append(k[b, :, :min(max(n, 0), S)])
        cache.append(1, k, v, counts=_ints(*cnt))
    K, _ = cache.get(1)
    lens = cache.lengths(1).tolist()
    assert lens == [sum(p.shape[1] for p in ps) for ps in parts]
    for b, ps in enumerate(parts):
        ref, _ = quantized(torch.cat(ps, 1))
        assert np.array_equal(K[b, :, :lens[b]].cpu().numpy(), ref)
        assert (K[b, :, lens[b]:] == 0).all() and (cache.positions(1)[b, :, lens[b]:] == -1).all()
    assert cache.get(0) is None and cache.seq_len == 0


@pytest.mark.parametrize("dtype", ALL)
def test_values_halfway_between_codes(L, dtype):
    """x / scale = k + 1/2 exactly, and the values beside those."""
    toks = []
    for m in range(4, 8) if dtype == torch.bfloat16 else range(16, 64):  # (2k + 1) m fits the type
        s = m * 2.0 ** -7
        for zero in (0, 3, 8):
            x = torch.arange(64, dtype=torch.float64) % 15 + 0.5 - zero
            x[0], x[1] = -zero, 15 - zero
            x = (x * s).to(dtype)
            assert torch.equal(x.double()[2:], ((torch.arange(64) % 15 + 0.5 - zero) * s).double()[2:])
            toks.append(x)
            up = x.float() * (1 + 2 * EPS[dtype])
            up[:2] = x[:2].float()
            toks += [up.to(dtype), (2 * x.float() - up).to(dtype)]
    k = torch.stack(toks).cuda()[None, None]
    cache = L.PackedKVCache(1, k.shape[2])
    cache.append(0, k, k.flip(2))
    a, b = cache.get(0)
    ref, _ = quantized(k)
    assert np.array_equal(a.cpu().numpy(), ref) and np.array_equal(b.flip(2).cpu().numpy(), ref)


def test_unusual_tokens(L):
    """All equal, all zero, one-sided, tiny, huge, NaN and infinite tokens."""
    D = 64
    x = torch.zeros(1, 1, 12, D, device="cuda")
    x[0, 0, 1] = 3.0
    x[0, 0, 2] = -2.5
    x[0, 0, 3] = torch.linspace(5.0, 6.0, D, device="cuda")
    x[0, 0, 4] = torch.linspace(-6.0, -5.0, D, device="cuda")
    x[0, 0, 5, 7] = 1e-6
    x[0, 0, 6] = torch.linspace(-1e-38, 1e-38, D, device="cuda")
    x[0, 0, 7] = torch.linspace(-1e30, 2e30, D, device="cuda")
    x[0, 0, 8, 3] = float("nan")
    x[0, 0, 9, 5] = float("inf")
    x[0, 0, 10, 5] = -float("inf")
    x[0, 0, 11] = torch.linspace(-0.5, 7.0, D, device="cuda")
    for dtype in ALL:
        y = x.to(dtype)
        cache = L.PackedKVCache(1, 12)
        cache.append(0, y, y)
        for got in cache.get(0):
            got = got[0, 0].cpu().numpy()
            ref, s = quantized(y[0, 0])
            bad = ~np.isfinite(s[:, 0])
            assert np.isnan(got[bad]).all() and bad.sum() >= 3
            assert np.array_equal(got[~bad], ref[~bad])
            step = np.abs(got - y[0, 0].float().cpu().numpy())[~bad]
            # half a step, and what the rounding of the scale takes from the range's end
            assert (step <= s[~bad] * (0.5 + 16 * 2.0 ** -8) + 16 * 2.0 ** -100).all()


# ---- attention: single tokens ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("T", [1, 2, 16, 31, 33, 500, 4099])
def test_decode_lengths(L, T, dtype, D):
    cache = L.PackedKVCache(1, T)
    cache.append(0, *_kv(2, 2, T, D, dtype, T))
    check(L, cache, _q(2, 8, 1, D, dtype, T + 1))


@pytest.mark.parametrize("G", [1, 3, 8, 9, 16, 20])
def test_decode_groups(L, G):
    cache = L.PackedKVCache(1, 777)
    cache.append(0, *_kv(1, 3, 777, 128, torch.float16, G))
    check(L, cache, _q(1, 3 * G, 1, 128, torch.float16, G))


@pytest.mark.parametrize("dtype", ALL)
def test_decode_ragged_with_empty_sequences(L, dtype):
    lens = (700, 0, 33, 1, 0, 1500, 64)
    cache = L.PackedKVCache(1, 1500)
    k, v = _kv(7, 2, 1500, 128, dtype, 3)
    cache.append(0, k, v, counts=_ints(*lens))
    q = _q(7, 8, 1, 128, dtype, 4)
    out = check(L, cache, q)
    assert (out[1] == 0).all() and (out[4] == 0).all()
    out = check(L, cache, q, counts=_ints(1, 1, 0, 1, 0, 1, 5))
    assert (out[2] == 0).all()


def test_many_sequences(L):
    """More sequences than a warp has lanes, more heads than blocks."""
    B = 70
    lens = [(37 * b) % 200 for b in range(B)]
    cache = L.PackedKVCache(1, 200)
    cache.append(0, *_kv(B, 16, 200, 64, torch.bfloat16, 5), counts=_ints(*lens))
    check(L, cache, _q(B, 32, 1, 64, torch.bfloat16, 6))
    check(L, cache, _q(B, 32, 1, 64, torch.bfloat16, 6), causal=True, window=20, prefix=_ints(*[b % 50 for b in range(B)]))


def test_scales_of_every_size(L):
    """Tokens whose K and V differ by orders of magnitude, zero tokens among
    them, and queries that fp16 could not hold as they are."""
    for dtype in (torch.float32, torch.bfloat16):
        k, v = (x.clone() for x in _kv(1, 2, 300, 64, dtype, 8))
        v *= torch.exp2(torch.randint(-30, 20, (1, 2, 300, 1), generator=_gen(1), device="cuda").float()).to(dtype)
        k *= torch.exp2(torch.randint(-20, 2, (1, 2, 300, 1), generator=_gen(2), device="cuda").float()).to(dtype)
        k[:, :, 10:20] = 0
        v[:, :, 15:30] = 0
        cache = L.PackedKVCache(1, 300)
        cache.append(0, k, v)
        for f in (1e-9, 1.0, 1e9):
            check(L, cache, _q(1, 4, 1, 64, dtype, 9) * f, scale=0.1 / f)
        cache = L.PackedKVCache(1, 300)
        cache.append(0, k, torch.zeros_like(v))
        assert (check(L, cache, _q(1, 4, 1, 64, dtype, 9)) == 0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("T", [2, 3, 7, 16, 40])
def test_few_tokens_whose_values_cancel(L, T, dtype):
    """Few rows and few tokens, V scales 2^10 apart: outputs near 0 show what
    an MMA cuts off.  With 16-bit queries half of V's codes are subnormals of
    which 2^-14 of a unit times the greatest p s_v among the 16 tokens of an
    MMA may be lost, in each of its 16 products: 2^-10 times the sum of those
    greatest ones beside the bound that the module's text derives."""
    for D, G, S, seed in ((64, 1, 1, 0), (128, 8, 2, 1), (64, 3, 1, 2), (128, 4, 4, 3)):
        k, v = _kv(4, 2, T, D, dtype, seed)
        v = v * torch.exp2(torch.randint(-5, 5, (4, 2, T, 1), generator=_gen(seed), device="cuda").float()).to(dtype)
        cache = L.PackedKVCache(1, T)
        cache.append(0, k, v)
        q = _q(4, 2 * G, S, D, dtype, seed + 5)
        ref, bound, _, _, _ = reference(cache, 0, q)
        x = torch.einsum("bhgsd,bhtd->bhgst", q.double().unflatten(1, (2, G)), cache.get(0)[0].double()) * D ** -0.5
        s_v = cache._layers[0].params[:, :, :T, 1].bitwise_left_shift(16).view(torch.float32).double()
        ps = torch.nn.functional.pad(torch.softmax(x, -1) * s_v[:, :, None, None], (0, -T % 16))
        cut = 2.0 ** -10 * ps.unflatten(-1, (-1, 16)).amax(-1).sum(-1) if dtype != torch.float32 else ps.sum(-1) * 0
        err = (cache.attend(0, q).double() - ref).abs() - cut.flatten(1, 2)[..., None]
        assert (err <= bound).all(), float((err / bound).max())


def test_nan_tokens_stay_behind_masks(L):
    """A NaN token reaches the queries that see it and no others."""
    k, v = (x.clone() for x in _kv(1, 2, 90, 64, torch.float16, 2))
    k[:, 0, 40] = float("nan")
    v[:, 1, 50] = float("inf")
    cache = L.PackedKVCache(1, 96)
    cache.append(0, k, v)
    q = _q(1, 4, 8, 64, torch.float16, 3)
    assert torch.isnan(cache.attend(0, q, causal=True)).all()
    out = cache.attend(0, q, causal=True, window=30)  # sees tokens 53 and later
    assert torch.isfinite(out).all()
    out = cache.attend(0, q, causal=True, window=46)  # the first queries see token 40 of head 0
    nan = torch.isnan(out).all(-1)
    at = torch.arange(82, 90, device="cuda")
    assert torch.equal(nan[0, :2], (at - 40 < 46).expand(2, -1)) and torch.equal(nan[0, 2:], (at - 50 < 46).expand(2, -1))
    # and in chunks
    k, v = (x.clone() for x in _kv(1, 2, 400, 64, torch.bfloat16, 2))
    k[:, 0, 140] = float("nan")
    v[:, 1, 150] = float("-inf")
    cache = L.PackedKVCache(1, 400)
    cache.append(0, k, v)
    q = _q(1, 4, 300, 64, torch.bfloat16, 3)
    p = torch.arange(100, 400, device="cuda")
    for window in (60, 0):
        nan = torch.isnan(cache.attend(0, q, causal=True, window=window)).all(-1)
        some = torch.isnan(cache.attend(0, q, causal=True, window=window)).any(-1)
        for heads, t in ((slice(0, 2), 140), (slice(2, 4), 150)):
            want = ((p >= t) & (p - t < (window or 1000))).expand(2, -1)
            assert torch.equal(nan[0, heads], want) and torch.equal(some[0, heads], want)


# ---- attention: chunks and score forms ---------------------------------------------------------------------------------

FORMS = {
    "plain": {},
    "causal": {"causal": True},
    "cap": {"causal": True, "softcap": 20.0},
    "bias": {"causal": True, "slopes": True},
    "both sides": {"slopes": True, "window": 9},
    "window": {"causal": True, "window": 33},
    "prefix": {"causal": True, "prefix": True},
    "all": {"causal": True, "softcap": 30.0, "slopes": True, "window": 50, "prefix": True},
}


def _form(name, B, Hq):
    f = dict(FORMS[name])
    if f.get("slopes"):
        f["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda").float() / Hq)
    if f.get("prefix"):
        f["prefix"] = _ints(*[(0, 40, 7, 500)[b % 4] for b in range(B)])
    return f


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("S", [1, 3, 40, 129])
@pytest.mark.parametrize("dtype", ALL)
def test_forms(L, dtype, S, form):
    B, H, G, D = 3, 2, 3, 128 if S % 2 else 64
    cache = L.PackedKVCache(1, 400)
    cache.append(0, *_kv(B, H, 200, D, dtype, S), counts=_ints(200, 11, 0))
    n = (S, max(1, S // 2), 0)
    cache.append(0, *_kv(B, H, S, D, dtype, S + 1), counts=_ints(*n))
    q = _q(B, H * G, S, D, dtype, S + 2)
    out = check(L, cache, q, counts=_ints(*n), **_form(form, B, H * G))
    assert (out[1, :, n[1]:] == 0).all() and (out[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,G,D,T,S", [(1, 8, 4, 128, 1100, 600), (2, 2, 1, 64, 515, 515), (1, 1, 7, 128, 2000, 333),
                                         (2, 3, 8, 64, 300, 17)])
def test_prompt_chunks(L, dtype, B, H, G, D, T, S):
    cache = L.PackedKVCache(1, T)
    cache.append(0, *_kv(B, H, T, D, dtype, T))
    q = _q(B, H * G, S, D, dtype, S)
    check(L, cache, q, causal=True)
    check(L, cache, q)
    check(L, cache, q, **_form("all", B, H * G))


@pytest.mark.parametrize("dtype,D", [(torch.float16, 128), (torch.bfloat16, 64)])
def test_chunks_with_rows_on_8_bytes(L, dtype, D):
    """Rows that only 8-byte copies can load, and the same rows on 16 bytes."""
    cache = L.PackedKVCache(1, 500)
    cache.append(0, *_kv(2, 2, 500, D, dtype, 1), counts=_ints(500, 301))
    wide = torch.randn(2, 6, 90, D + 4, generator=_gen(2), device="cuda").to(dtype)
    q = wide[..., 4:]
    assert q.data_ptr() % 16 == 8 and q.stride(2) % 8 == 4
    out = check(L, cache, q, causal=True)
    assert torch.equal(out, cache.attend(0, q.contiguous(), causal=True))


@pytest.mark.parametrize("G,S", [(300, 1), (129, 3), (1000, 2), (17, 1), (7, 61)])
def test_many_query_heads(L, G, S):
    """Groups that are no power of two and larger than a tile."""
    cache = L.PackedKVCache(1, 700)
    cache.append(0, *_kv(1, 2, 700, 64, torch.float16, 3))
    slopes = torch.rand(2 * G, generator=_gen(4), device="cuda") * 0.1
    check(L, cache, _q(1, 2 * G, S, 64, torch.float16, 5), causal=True, slopes=slopes, window=333)


def test_scales_of_every_size_in_chunks(L):
    """As for single tokens, but no scale differs by more than 2^16 within 128
    tokens: P is kept beside the greatest V scale of a tile there."""
    for dtype in (torch.float16, torch.bfloat16):
        k, v = (x.clone() for x in _kv(1, 2, 700, 64, dtype, 8))
        v *= torch.exp2(torch.randint(-6, 6, (1, 2, 700, 1), generator=_gen(1), device="cuda").float()).to(dtype)
        k *= torch.exp2(torch.randint(-10, 2, (1, 2, 700, 1), generator=_gen(2), device="cuda").float()).to(dtype)
        k[:, :, 10:20] = 0
        v[:, :, 15:30] = 0
        v[:, :, 256:400] = 0  # a whole tile of zeros
        cache = L.PackedKVCache(1, 700)
        cache.append(0, k, v)
        q = _q(1, 4, 100, 64, dtype, 9)
        check(L, cache, q, causal=True)
        check(L, cache, q * 30, causal=True, scale=0.4)  # peaked: references are raised again and again
        check(L, cache, q, softcap=5.0, window=300)


@pytest.mark.parametrize("dtype,D", [(torch.float16, 128), (torch.bfloat16, 64)])
def test_scores_that_rise_along_the_tokens(L, dtype, D):
    """Each 32 tokens beat those before by more than a reference has room
    for, so that both halves of every step raise it."""
    T, S = 400, 70
    k, v = (x.clone() for x in _kv(2, 2, T, D, dtype, 1))
    up = (torch.arange(T, device="cuda") // 32).double() / 4
    k = (torch.randn(D, generator=_gen(3), device="cuda") * up[:, None]).to(dtype).expand(2, 2, T, D)
    cache = L.PackedKVCache(1, T)
    cache.append(0, k, v, counts=_ints(T, 333))
    q = _q(2, 8, S, D, dtype, 4)
    for scale in (1.0, -1.0, 4.0):
        for kw in ({}, {"causal": True}, {"causal": True, "window": 150}, {"softcap": 300.0}):
            check(L, cache, q, scale=scale, **kw)
    slopes = torch.linspace(0.3, 2.0, 8, device="cuda")
    check(L, cache, q, causal=True, slopes=slopes, scale=0.1)
    cache.evict(0, 200)
    check(L, cache, q, causal=True, scale=1.0)
    # the weight of the halves of one step: 32 tokens at 0, 32 a factor 2^9 .. 2^14 above, and so on
    v = torch.ones(1, 1, T, D, device="cuda").to(dtype)
    v[..., 1::2] *= ((torch.arange(T, device="cuda") // 32) % 2)[:, None].to(dtype)
    k = torch.zeros(1, 1, T, D, device="cuda", dtype=dtype)
    k[..., 0] = (torch.arange(T, device="cuda") // 32).to(dtype)
    q = torch.zeros(1, 2, S, D, device="cuda", dtype=dtype)
    q[..., 0] = torch.linspace(6.5, 9.5, 2 * S, device="cuda").view(1, 2, S).to(dtype)
    cache = L.PackedKVCache(1, T)
    cache.append(0, k, v)
    for kw in ({}, {"causal": True}, {"softcap": 300.0}):  # the cap has every tile go the masked way
        check(L, cache, q, scale=1.0, **kw)


@pytest.mark.parametrize("S", [1, 40])
@pytest.mark.parametrize("dtype", ALL)
def test_large_caps(L, dtype, S):
    """A cap far above the scores changes them as its formula says, and loses
    no bits of them: tanh of a small argument is good to 2^-23 of itself, a score x then to 2^-21 |x|
    on top of dx = 12 * 2^-22 a, and |x| <= a: dx <= 14 / 12 of what it is
    without a cap.  A cap of 1000 or more changes scores up to 20 by less than
    20^3 / (3 * 1000^2) = 0.003, so probabilities in the bound by 0.6 %:
    1.2 > 14 / 12 * 1.006 covers both."""
    B, H, G, D, T = 2, 2, 4, 64, 700
    cache = L.PackedKVCache(1, T)
    cache.append(0, *_kv(B, H, T, D, dtype, 1), counts=_ints(T, 333))
    q = _q(B, H * G, S, D, dtype, 2)
    _, bound, _, mb, _ = reference(cache, 0, q, causal=True)
    for cap in (1e3, 1e4, 1e5, 1e6, 1e7, 1e9, 1e15, 1e30):
        ref, _, m, _, _ = reference(cache, 0, q, causal=True, softcap=cap)
        cache.attention_mass(0).zero_()
        out = cache.attend(0, q, causal=True, softcap=cap, accumulate=True)
        err = (out.double() - ref).abs()
        assert (err <= 1.2 * bound).all(), (cap, float((err / bound).max()))
        err = (cache.attention_mass(0).double() - m).abs()
        assert (err <= 1.2 * mb).all(), (cap, float((err / mb).max()))


def test_probabilities_of_chunks_are_rounded_once(L):
    """32 tokens, then one whose score passes the reference's headroom in the
    same step: the first 32 keep one rounding each.  They have the same
    probability p and the value 1, the rest the value 0, so out = 32 p: off by
    2^-11 for P, 2^-11 for the output, and 2 (dx + 2^-20) with dx = 12 * 2^-22
    times a score of at most 9.1."""
    S, T, D = 256, 64, 64
    k = torch.zeros(1, 1, T, D, device="cuda", dtype=torch.float16)
    k[..., 32, :2] = 1
    v = torch.zeros(1, 1, T, D, device="cuda", dtype=torch.float16)
    v[..., :32, :] = 1
    cache = L.PackedKVCache(1, T)
    cache.append(0, k, v)
    q = torch.zeros(1, 8, S, D, device="cuda", dtype=torch.float16)
    q[..., 0] = torch.linspace(6.5, 8.9, 8 * S, device="cuda").view(1, 8, S)
    q[..., 1] = torch.rand(1, 8, S, generator=_gen(1), device="cuda") * 0.1
    kv, vv = (x.double() for x in cache.get(0))
    x = torch.einsum("hsd,td->hst", q[0].double(), kv[0, 0])
    assert 6.4 < x.amax(-1).min() and x.max() < 9.1
    ref = torch.softmax(x, -1) @ vv[0, 0]
    out = cache.attend(0, q, scale=1.0, slopes=torch.zeros(8, device="cuda"))[0].double()
    err = ((out - ref) / ref).abs().max().item()
    assert err <= 2 * 2.0 ** -11 + 2 * (12 * 2.0 ** -22 * 9.1 + 2.0 ** -20), err * 2.0 ** 11


def test_windows_and_prefixes_of_any_size(L):
    cache = L.PackedKVCache(1, 300)
    cache.append(0, *_kv(2, 2, 300, 64, torch.bfloat16, 8), counts=_ints(300, 77))
    for S in (1, 50):
        q = _q(2, 8, S, 64, torch.bfloat16, S)
        for window in (1, 2, 64, 128, 299, 300, 2 ** 30):
            for prefix in (None, _ints(0, -5), _ints(2 ** 31 - 1, 1), _ints(130, 64)):
                for causal in (True, False):
                    check(L, cache, q, causal=causal, window=window, prefix=prefix)


def test_query_layouts_give_the_same(L):
    cache = L.PackedKVCache(1, 256)
    cache.append(0, *_kv(2, 2, 256, 64, torch.bfloat16, 1))
    q = _q(2, 4, 5, 64, torch.bfloat16, 2)
    ref = cache.attend(0, q, causal=True)
    assert torch.equal(cache.attend(0, q.contiguous(), causal=True), ref)
    wide = torch.zeros(2, 4, 5, 131, device="cuda", dtype=torch.bfloat16)
    wide[..., 1:65] = q
    assert torch.equal(cache.attend(0, wide[..., 1:65], causal=True), ref)  # rows on odd addresses
    assert torch.equal(cache.attend(0, q.transpose(2, 3).contiguous().transpose(2, 3), causal=True), ref)
    one = _q(2, 1, 5, 64, torch.bfloat16, 3).expand(2, 4, 5, 64)  # broadcast heads
    assert torch.equal(cache.attend(0, one, causal=True), cache.attend(0, one.contiguous(), causal=True))
    k = torch.randn(2, 1, 9, 64, device="cuda").expand(2, 2, 9, 64)
    a, b = L.PackedKVCache(1, 9), L.PackedKVCache(1, 9)
    a.append(0, k, k), b.append(0, k.contiguous(), k.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a.get(0), b.get(0)))


# ---- collected weight and eviction ---------------------------------------------------------------------------------------

def expected_evict(positions, mass, n, nxt, keep, recent, sinks):
    """Slots that end up in 0 .. keep - 1, for one head."""
    if n <= keep:
        return list(range(n))

    def key(t):
        p, m = positions[t], mass[t]
        safe = p >= nxt - recent or p < sinks
        return (not safe, not math.isnan(m), -max(m, 0.0) if not math.isnan(m) else 0.0, t)

    kept = set(sorted(range(n), key=key)[:keep])
    late = iter([t for t in range(keep, n) if t in kept])
    return [t if t in kept else next(late) for t in range(keep)]


def check_evict(cache, keep, recent=0, sinks=0, layer=0):
    st = cache._layers[layer]
    K, V = cache.get(layer)
    pos, mass, lens = cache.positions(layer).cpu(), cache.attention_mass(layer).cpu(), cache.lengths(layer).tolist()
    nxt = st.state[st.B:2 * st.B].tolist()
    cache.evict(layer, keep, recent=recent, sinks=sinks)
    K2, V2 = cache.get(layer)
    pos2, mass2 = cache.positions(layer).cpu(), cache.attention_mass(layer).cpu()
    assert cache.lengths(layer).tolist() == [min(n, keep) for n in lens]
    assert st.state[st.B:2 * st.B].tolist() == nxt
    assert st.state[2 * st.B].item() == 0  # the ticket is back
    for b in range(st.B):
        for h in range(st.H):
            src = expected_evict(pos[b, h].tolist(), mass[b, h].tolist(), lens[b], nxt[b], keep, recent, sinks)
            m = len(src)
            assert pos2[b, h, :m].tolist() == pos[b, h, src].tolist(), (b, h)
            assert torch.equal(mass2[b, h, :m].view(torch.int32), mass[b, h, src].view(torch.int32))
            assert torch.equal(K2[b, h, :m], K[b, h, src]) and torch.equal(V2[b, h, :m], V[b, h, src])
    whole = st.positions.cpu()
    for b in range(st.B):
        assert (whole[b, :, min(lens[b], keep):] == -1).all() and (st.mass[b, :, min(lens[b], keep):] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,keep,recent,sinks", [(10, 9, 0, 0), (10, 1, 0, 0), (40, 20, 20, 0), (100, 37, 5, 4),
                                                 (1500, 1024, 100, 4), (1500, 1400, 0, 7), (5000, 33, 8, 0),
                                                 (5000, 3000, 2996, 4), (3000, 2999, 1, 0)])
def test_evict(L, T, keep, recent, sinks, D):
    cache = L.PackedKVCache(1, T + 5)
    lens = (T, max(1, T // 2), keep)
    cache.append(0, *_kv(3, 2, T, D, torch.bfloat16, T), counts=_ints(*lens))
    live = torch.arange(T, device="cuda") < _ints(*lens)[:, None, None]
    m = torch.exp(3 * torch.randn(3, 2, T, generator=_gen(T), device="cuda"))
    cache.attention_mass(0).copy_(torch.where(live, m, 0.0))
    check_evict(cache, keep, recent, sinks)


def test_evict_ties_and_odd_masses(L):
    cache = L.PackedKVCache(1, 3000)
    cache.append(0, *_kv(1, 3, 3000, 64, torch.float16, 1))
    m = torch.zeros(1, 3, 3000, device="cuda")
    m[0, 1, ::3] = 0.25  # few different values: ties everywhere
    m[0, 2, 5] = float("nan")
    m[0, 2, 7] = -float("nan")
    m[0, 2, 2999] = float("inf")
    m[0, 2, 11] = 1e-45
    m[0, 2, 13] = -1.0  # counts as 0
    m[0, 2, 2000] = 3.4e38
    cache.attention_mass(0).copy_(m)
    check_evict(cache, 1100)
    check_evict(cache, 700)   # of a cache whose slots are out of order
    check_evict(cache, 40, recent=9, sinks=3)
    check_evict(cache, 2)
    cache.append(0, *_kv(1, 3, 100, 64, torch.float16, 2))
    check_evict(cache, 100, recent=50)


def test_evict_more_tokens_than_shared_memory_holds(L):
    T, keep = 60001, 55000
    cache = L.PackedKVCache(1, T)
    cache.append(0, *_kv(1, 1, T, 64, torch.float16, 1))
    cache.attention_mass(0).copy_(torch.exp(3 * torch.randn(1, 1, T, generator=_gen(1), device="cuda")))
    check_evict(cache, keep, recent=50, sinks=4)
    check(L, cache, _q(1, 4, 30, 64, torch.float16, 2), causal=True, window=40000)


def test_masks_go_by_position_after_eviction(L):
    for dtype in ALL:
        B, H, G, D = 2, 2, 4, 128
        cache = L.PackedKVCache(1, 500)
        cache.append(0, *_kv(B, H, 400, D, dtype, 1), counts=_ints(400, 90))
        cache.attend(0, _q(B, H * G, 1, D, dtype, 2), accumulate=True)
        cache.evict(0, 150, recent=10, sinks=4)
        for S in (1, 7, 60):
            cache.append(0, *_kv(B, H, S, D, dtype, S))
            for form in FORMS:
                check(L, cache, _q(B, H * G, S, D, dtype, S + 1), **_form(form, B, H * G))
            cache.attention_mass(0).abs_()  # whatever the checks added: weights
            check_evict(cache, 150, recent=S, sinks=4)


def test_distances_at_far_positions(L):
    """Positions past 2^24, where fp32 has no more odd numbers: as after
    so many tokens through a cache that evicts."""
    far = 2 ** 25 + 1
    for dtype in ALL:
        cache = L.PackedKVCache(1, 300)
        cache.append(0, *_kv(2, 2, 300, 64, dtype, 1), counts=_ints(300, 133))
        st = cache._layers[0]
        st.state[2:4] += far
        st.state[6] = 1  # slots are not positions any more
        st.positions.add_(far * (st.positions >= 0))
        slopes = torch.exp2(-torch.arange(1, 9, device="cuda").float())
        for S in (1, 70):
            q = _q(2, 8, S, 64, dtype, 2)
            for kw in ({}, {"causal": True}, {"causal": True, "window": 77}, {"causal": True, "softcap": 20.0}):
                check(L, cache, q, slopes=slopes, **kw)


def test_row_that_sees_nothing_after_eviction(L):
    """Everything within the window was evicted: zeros, and no weight."""
    cache = L.PackedKVCache(1, 64)
    cache.append(0, *_kv(1, 1, 64, 64, torch.float16, 1))
    m = torch.arange(64, 0, -1, device="cuda").float().view(1, 1, 64)
    cache.attention_mass(0).copy_(m)
    cache.evict(0, 8)  # positions 0 .. 7 stay
    q = _q(1, 2, 3, 64, torch.float16, 2)
    assert (check(L, cache, q, causal=True, window=10) == 0).all()
    check(L, cache, q, causal=True, window=10, prefix=_ints(3))


# ---- together ------------------------------------------------------------------------------------------------------------

def test_decode_loop_with_a_budget(L):
    """Prompt, then single tokens: append, attend with collected weight, evict."""
    B, H, G, D, keep = 2, 2, 4, 128, 96
    cache = L.PackedKVCache(2, 300)
    for layer in range(2):
        cache.append(layer, *_kv(B, H, 150, D, torch.bfloat16, layer), counts=_ints(150, 60))
        cache.attend(layer, _q(B, H * G, 150, D, torch.bfloat16, layer), causal=True, counts=_ints(150, 60),
                     accumulate=True)
        check_evict(cache, keep, recent=16, sinks=4, layer=layer)
    for step in range(50):
        for layer in range(2):
            seed = 100 + 2 * step + layer
            cache.append(layer, *_kv(B, H, 1, D, torch.bfloat16, seed))
            q = _q(B, H * G, 1, D, torch.bfloat16, seed)
            if step % 10 == 0:
                check(L, cache, q, layer=layer, causal=True)
            else:
                cache.attend(layer, q, causal=True, accumulate=True)
            if step % 10 == 5:
                check_evict(cache, keep, recent=16, sinks=4, layer=layer)
            else:
                cache.evict(layer, keep, recent=16, sinks=4)
    assert cache.lengths(1).tolist() == [96, 96] and cache.seq_len == 96
    cache.check(0), cache.check(1)
    cache.reset()
    assert cache.seq_len == 0 and cache.lengths(0).tolist() == [0, 0]
    cache.append(0, *_kv(B, H, 5, D, torch.bfloat16, 1))
    assert cache.positions(0)[0, 0].tolist() == [0, 1, 2, 3, 4]
    check(L, cache, _q(B, H * G, 2, D, torch.bfloat16, 1), causal=True, window=2)


def test_captured_loop_equals_the_eager_one(L):
    B, H, G, D, keep = 2, 2, 4, 64, 70
    caches = [L.PackedKVCache(1, 160) for _ in range(2)]
    for c in caches:
        c.append(0, *_kv(B, H, 60, D, torch.float16, 0), counts=_ints(60, 31))
    ins = [(*_kv(B, H, 1, D, torch.float16, 10 + i), _q(B, H * G, 1, D, torch.float16, 50 + i)) for i in range(30)]
    k, v, q = (x.clone() for x in ins[0])

    def step(c, k, v, q):
        c.append(0, k, v)
        o = c.attend(0, q, causal=True, softcap=30.0, accumulate=True)
        c.evict(0, keep, recent=8, sinks=2)
        return o

    snapshot = [t.clone() for t in (caches[0]._layers[0].k_codes, caches[0]._layers[0].v_codes,
                                    caches[0]._layers[0].params, caches[0]._layers[0].positions,
                                    caches[0]._layers[0].mass, caches[0]._layers[0].state)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(caches[0], k, v, q)  # warm-up, taken back below
    side.synchronize()
    st = caches[0]._layers[0]
    for t, s in zip((st.k_codes, st.v_codes, st.params, st.positions, st.mass, st.state), snapshot):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], k, v, q)
    for x in ins:
        for t, s in zip((k, v, q), x):
            t.copy_(s)
        graph.replay()
        ref = step(caches[1], *x)
        # the capture splits the work for the whole room: other partial sums
        assert (out.float() - ref.float()).abs().max() <= 4 * 2.0 ** -11 * ref.float().abs().max()
    assert torch.equal(caches[0].lengths(0), caches[1].lengths(0))
    n = caches[1].seq_len
    assert torch.equal(caches[0].positions(0)[:, :, :n], caches[1].positions(0))
    assert caches[0].dropped(0).item() == 0
    del graph


def test_replayed_appends_stop_at_the_room(L):
    cache = L.PackedKVCache(1, 40)
    k, v = _kv(2, 1, 7, 64, torch.float16, 0)
    cnt = _ints(7, 3)
    cache.append(0, k, v, counts=cnt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, k, v, counts=cnt)
    for _ in range(12):
        graph.replay()
    cap = cache._layers[0].cap
    assert cap == 64 and cache.lengths(0).tolist() == [64, 39]
    assert cache.dropped(0).item() == 13 * 7 - 64
    assert cache.positions(0)[0, 0, :40].tolist() == list(range(40))
    out = cache.attend(0, _q(2, 2, 1, 64, torch.float16, 1))
    assert torch.isfinite(out).all()
    del graph


def test_replayed_evictions_start_with_little(L):
    """Captured while nothing had to go; the appends between replays are eager."""
    cache = L.PackedKVCache(1, 64)
    cache.append(0, *_kv(2, 1, 10, 64, torch.float16, 0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.evict(0, 20, recent=20)
    assert cache.seq_len == 64
    for n in range(4):
        cache.append(0, *_kv(2, 1, 9, 64, torch.float16, n))
        graph.replay()
        assert cache.lengths(0).tolist() == [min(20, 10 + 9 * (n + 1))] * 2
    assert sorted(cache.positions(0)[1, 0, :20].tolist()) == list(range(26, 46))
    cache.reset()
    assert cache.seq_len == 0
    del graph


def test_replays_after_a_reset(L):
    """A decode step captured once; each request resets, appends its prompt and replays."""
    B, H, D, room, keep = 2, 2, 64, 160, 40
    cache = L.PackedKVCache(1, room)
    k, v = (x.clone() for x in _kv(B, H, 1, D, torch.float16, 0))
    q = _q(B, 4, 1, D, torch.float16, 1)
    cache.append(0, k, v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, k, v)
        cache.attend(0, q, causal=True, accumulate=True)
    for request in range(2):
        cache.reset()
        assert cache.seq_len == 0
        graph.replay()  # the host sees nothing of it
        assert cache.seq_len == room and cache.lengths(0).tolist() == [1, 1]
        cache.reset()
        twin = L.PackedKVCache(1, room)
        prompt, counts = _kv(B, H, 30, D, torch.float16, 10 + request), _ints(30, 17)
        for c in (cache, twin):
            c.append(0, *prompt, counts=counts)
        for step in range(25):
            new = _kv(B, H, 1, D, torch.float16, 100 * request + step)
            k.copy_(new[0]), v.copy_(new[1])
            graph.replay()
            twin.append(0, *new)
            twin.attend(0, q, causal=True, accumulate=True)
        n = 55
        assert cache.lengths(0).tolist() == twin.lengths(0).tolist() == [n, n - 13]
        assert cache.seq_len == room
        for a, b in zip(cache.get(0), twin.get(0)):
            assert torch.equal(a[:, :, :n], b) and not a[:, :, n:].any()
        assert torch.equal(cache.positions(0)[:, :, :n], twin.positions(0))
        cache.attention_mass(0).mul_(0.5)  # reaches every token
        assert (cache.attention_mass(0)[:, :, :n] > 0).sum().item() == 2 * (2 * n - 13)
        check_evict(cache, keep, recent=4)
        assert cache.lengths(0).tolist() == [keep, keep]
        cache.append(0, *prompt, counts=counts)
        check(L, cache, q, causal=True)
    # a captured reset is the replay's
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        cache.reset()
    assert cache.seq_len == room and cache.lengths(0).tolist() != [0, 0]
    assert cache.get(0)[0].any()
    again.replay()
    assert cache.lengths(0).tolist() == [0, 0] and not cache.get(0)[0].any()
    del graph, again


def test_first_chunk_is_not_captured(L):
    """Its buffers would be made, and emptied, by every replay."""
    cache = L.PackedKVCache(2, 64)
    k, v = _kv(1, 1, 3, 64, torch.float16, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        k2 = k + 0
        for n in (3, 0):
            with pytest.raises(RuntimeError, match="capture"):
                cache.append(0, k[:, :, :n], v[:, :, :n])
    assert cache.get(0) is None
    cache.append(0, k[:, :, :0], v[:, :, :0])  # makes room, as the message says
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, k, v)
    for n in (3, 6):
        graph.replay()
        assert cache.lengths(0).tolist() == [n]
    del graph, k2


def test_replayed_tokens_past_max_seq_len_can_be_read(L):
    """The room is max_seq_len rounded up to 32; replays may fill all of it."""
    cache, twin = L.PackedKVCache(1, 40), L.PackedKVCache(1, 70)
    k, v = _kv(2, 1, 7, 64, torch.float16, 0)
    cnt = _ints(7, 3)
    for c in (cache, twin):
        c.append(0, k, v, counts=cnt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(0, k, v, counts=cnt)
    for _ in range(8):
        graph.replay()
        twin.append(0, k, v, counts=cnt)
    n = cache.lengths(0)
    assert n.tolist() == [63, 27] and cache.seq_len >= 63
    for a, b in zip((*cache.get(0), cache.positions(0)), (*twin.get(0), twin.positions(0))):
        assert torch.equal(a[:, :, :63], b[:, :, :63])
    cache.attend(0, _q(2, 2, 1, 64, torch.float16, 1), accumulate=True)
    assert (cache.attention_mass(0) > 0).sum((1, 2)).tolist() == n.tolist()
    with pytest.raises(ValueError, match="fit"):
        cache.append(0, *_kv(2, 1, 65, 64, torch.float16, 0))
    del graph


def test_replayed_attention_outgrows_its_capture(L):
    """Captured with few tokens, replayed with many: grids are made for few."""
    for S, dtype in ((1, torch.bfloat16), (30, torch.bfloat16), (30, torch.float32)):
        cache, twin = L.PackedKVCache(1, 3000), L.PackedKVCache(1, 3000)
        for c in (cache, twin):
            c.append(0, *_kv(2, 2, 40, 64, dtype, 0), counts=_ints(40, 33))
        q = _q(2, 4, S, 64, dtype, 1)
        cache.attend(0, q, causal=True, accumulate=True)
        torch.cuda.synchronize()
        cache.attention_mass(0).zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = cache.attend(0, q, causal=True, accumulate=True)
        for c in (cache, twin):
            c.append(0, *_kv(2, 2, 2900, 64, dtype, 2), counts=_ints(2900, 1700))
        graph.replay()
        ref, bound, m, mb, _ = reference(twin, 0, q, causal=True)
        assert ((out.double() - ref).abs() <= bound).all()
        assert ((cache.attention_mass(0).double() - m).abs() <= mb).all()
        cache.check(0)
        del graph


def test_collected_weight_without_kept_scores(L):
    """So much room that the scores of a call would take more than 256 MB."""
    cache = L.PackedKVCache(1, 2 ** 22 + 64)
    cache.append(0, *_kv(1, 1, 3000, 64, torch.bfloat16, 0))
    for kw in ({}, dict(softcap=20.0, window=700)):
        check(L, cache, _q(1, 16, 1, 64, torch.bfloat16, 1), **kw)


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("dtype,D", [(torch.float16, 64), (torch.bfloat16, 128)])
def test_collected_weight_of_one_or_two_row_tiles(L, dtype, D, form):
    """Chunks of one, two and three tiles of 128 rows side by side, more tiles
    of tokens than SMs: a row tile's sums may run ahead of the other's."""
    B, H, G, S, T = 6, 4, 4, 70, 3000
    n = (20, 40, 5, 64, 70, 1)
    cache = L.PackedKVCache(1, T)
    cache.append(0, *_kv(B, H, T, D, dtype, 1), counts=_ints(T, 2500, 2999, 130, 1700, 2000))
    q = _q(B, H * G, S, D, dtype, 2)
    kw = dict(_form(form, B, H * G), counts=_ints(*n))
    check(L, cache, q, **kw)
    mass = []
    for _ in range(4):
        cache.attention_mass(0).zero_()
        cache.attend(0, q, accumulate=True, **kw)
        mass.append(cache.attention_mass(0).clone())
    assert all(torch.equal(m, mass[0]) for m in mass)


def test_whole_heads_and_cut_ones(L):
    """Lengths around those where a block takes a whole head, and scales of either sign."""
    for T in (480, 511, 512, 513, 600, 1100):
        cache = L.PackedKVCache(1, T)
        cache.append(0, *_kv(2, 3, T, 128, torch.float16, T), counts=_ints(T, T // 2))
        for scale in (None, 0.0, -0.1):
            check(L, cache, _q(2, 6, 1, 128, torch.float16, 1), scale=scale)
            check(L, cache, _q(2, 6, 40, 128, torch.float16, 1), scale=scale, causal=True)


@pytest.mark.parametrize("dtype,S", [(torch.bfloat16, 1), (torch.float32, 5)])
def test_split_follows_the_length(L, dtype, S):
    """The work of a cache that grew is split as that of one that began as long."""
    q = _q(1, 8, S, 64, dtype, 1)
    grown = L.PackedKVCache(1, 9000)
    for n, total in ((300, 300), (300, 600), (4200, 4800), (4000, 8800)):
        grown.append(0, *_kv(1, 8, n, 64, dtype, total))
        out = grown.attend(0, q, accumulate=True)
        fresh = L.PackedKVCache(1, 9000)
        fresh.append(0, *_kv(1, 8, total, 64, dtype, 0))
        fresh.attend(0, q, accumulate=True)
        (_, need, form), = fresh._layers[0].forms.values()
        used = list(grown._layers[0].forms.values())[-1]
        assert used[1] == need and used[2].bound == form.bound
        assert torch.isfinite(out).all()


def test_scale_as_a_tensor_is_read_at_each_call(L):
    cache = L.PackedKVCache(1, 100)
    cache.append(0, *_kv(1, 2, 100, 64, torch.float16, 0))
    q = _q(1, 4, 1, 64, torch.float16, 1)
    scale = torch.tensor(0.1)
    a = cache.attend(0, q, scale=scale)
    assert torch.equal(a, cache.attend(0, q, scale=scale.item()))
    scale.fill_(0.3)
    assert torch.equal(cache.attend(0, q, scale=scale), cache.attend(0, q, scale=scale.item()))
    assert torch.equal(cache.attend(0, q, window=torch.tensor(7)), cache.attend(0, q, window=7))


def test_two_calls_at_once_and_other_streams(L):
    cache = L.PackedKVCache(1, 3000)
    cache.append(0, *_kv(4, 4, 3000, 128, torch.bfloat16, 0))
    qs = [_q(4, 16, 1, 128, torch.bfloat16, i) for i in range(8)]
    ref = [cache.attend(0, q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 4]):
            outs.append(cache.attend(0, q))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, ref))


def test_results_do_not_change_from_run_to_run(L):
    def once():
        cache = L.PackedKVCache(1, 2500)
        cache.append(0, *_kv(2, 2, 2500, 128, torch.bfloat16, 0))
        a = cache.attend(0, _q(2, 8, 1, 128, torch.bfloat16, 1), accumulate=True)
        b = cache.attend(0, _q(2, 8, 300, 128, torch.bfloat16, 2), causal=True, accumulate=True)
        cache.evict(0, 1000, recent=10)
        return a, b, cache.attention_mass(0).clone(), cache.positions(0).clone()

    first = once()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, once()))


def test_offsets_past_32_bits(L):
    """64 heads of 2^19 tokens of room: codes of the last heads lie past 2^31 bytes."""
    room = 2 ** 19 + 32 * 7
    cache = L.PackedKVCache(1, room)
    cache.append(0, *_kv(8, 8, 50, 128, torch.bfloat16, 0))
    k, v = cache.get(0)
    ref, _ = quantized(_kv(8, 8, 50, 128, torch.bfloat16, 0)[0])
    assert np.array_equal(k.cpu().numpy(), ref)
    check(L, cache, _q(8, 16, 1, 128, torch.bfloat16, 1))
    check(L, cache, _q(8, 16, 20, 128, torch.bfloat16, 1), causal=True)
    cache.attention_mass(0).abs_()
    check_evict(cache, 20, recent=4)


def test_agrees_with_the_byte_cache(L):
    """The same tokens in QuantizedKVCache with the reference's 4-bit
    quantizer: fp32 codes are taken in the same way, but for the scale's
    rounding to bf16, so values differ by half a step of 2^-8 at most, or by a
    step where that moves a value over a border."""
    k, v = _kv(2, 2, 333, 128, torch.float32, 0)
    byte = L.QuantizedKVCache(1, L.PerTokenKVCacheQuantizer(4, symmetric=False))
    fk, fv = byte.update(0, k, v)
    cache = L.PackedKVCache(1, 333)
    pk, pv = cache.update(0, k, v)
    for a, b, x in ((fk, pk, k), (fv, pv, v)):
        step = (x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)) / 15
        assert ((a - b).abs() <= step * (1 + 16 * 2.0 ** -8)).all()
        assert ((a - b).abs() > step / 2).float().mean() < 0.03


# ---- refusals ------------------------------------------------------------------------------------------------------------

def test_check_reports_a_wait_that_ran_out(L):
    """The status word as a kernel would leave it, set from the host."""
    from llm_quant_b200 import _C
    cache = L.PackedKVCache(1, 32)
    cache.append(0, *_kv(2, 2, 20, 64, torch.float16, 0))
    cache.check(0)
    cache._layers[0].state[-1] = _C.ETIMEOUT
    for _ in range(2):  # stays until the cache is emptied
        with pytest.raises(_C.LQError, match="ran out") as e:
            cache.check(0)
        assert e.value.status == _C.ETIMEOUT
    cache.reset()
    cache.check(0)


def test_refusals_on_the_device(L):
    cache = L.PackedKVCache(1, 32)
    k, v = _kv(2, 2, 20, 64, torch.float16, 0)
    with pytest.raises(RuntimeError, match="empty"):
        cache.attend(0, _q(2, 2, 1, 64, torch.float16, 0))
    with pytest.raises(RuntimeError, match="empty"):
        cache.evict(0, 3)
    with pytest.raises(RuntimeError, match="empty"):
        cache.lengths(0)
    cache.append(0, k, v)
    with pytest.raises(ValueError, match="do not fit"):
        cache.append(0, k, v)
    with pytest.raises(RuntimeError, match="new"):
        cache.append(0, k[:1], v[:1])
    with pytest.raises(RuntimeError, match="both"):
        cache.append(0, k, v[:, :, :3])
    with pytest.raises(TypeError):
        cache.append(0, k, v.float())
    with pytest.raises(TypeError):
        cache.append(0, k.int(), v.int())
    with pytest.raises(ValueError, match="counts"):
        cache.append(0, k[:, :, :2], v[:, :, :2], counts=torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="counts"):
        cache.append(0, k[:, :, :2], v[:, :, :2], counts=torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="counts"):
        cache.append(0, k[:, :, :2], v[:, :, :2], counts=_ints(1, 1, 1))
    q = _q(2, 4, 1, 64, torch.float16, 0)
    for bad in (q[:, :3], q[:1], q[..., :32], q[0], q[:, :0]):
        with pytest.raises(RuntimeError, match="match"):
            cache.attend(0, bad)
    with pytest.raises(TypeError):
        cache.attend(0, q.long())
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.attend(0, q.cpu())
    for kw in ({"softcap": -1.0}, {"softcap": float("nan")}, {"softcap": float("inf")}, {"softcap": 1e-30}, {"window": -1}, {"window": 2 ** 30 + 1},
               {"slopes": torch.ones(4, device="cuda", dtype=torch.float16)}, {"slopes": torch.ones(3, device="cuda")},
               {"slopes": torch.ones(8, device="cuda")[::2]}, {"prefix": torch.ones(2, device="cuda")},
               {"prefix": 4}, {"counts": [1, 1]}):
        with pytest.raises(ValueError):
            cache.attend(0, q, **kw)
    for a in ((0,), (-1,), (4, 5), (4, 2, 3), (4, -1), (4, 0, -1)):
        with pytest.raises(ValueError):
            cache.evict(0, *a)
    with pytest.raises(TypeError):
        cache.get(0, torch.int8)
    with pytest.raises(ValueError, match="head dim"):
        L.PackedKVCache(1, 8).append(0, torch.zeros(1, 1, 1, 96, device="cuda"), torch.zeros(1, 1, 1, 96, device="cuda"))
    with pytest.raises(ValueError, match="fit"):
        L.PackedKVCache(1, 8).append(0, k, v)
    assert cache.lengths(0).tolist() == [20, 20]
    # empty work is no work
    cache.append(0, k[:, :, :0], v[:, :, :0])
    assert cache.attend(0, q[:, :, :0]).shape == (2, 4, 0, 64)
    cache.evict(0, 20)
    assert cache.lengths(0).tolist() == [20, 20]
    check(L, cache, q)
