"""CPU-side checks of the 4-bit KV cache: what PackedKVCache and the lq_kv4_*
entry points refuse before any launch (no GPU needed)."""

import ctypes

import pytest
import torch

import llm_quant_b200 as L


@pytest.fixture(scope="module")
def lib():
    from llm_quant_b200 import _C, build
    build.build()
    return _C.lib()


def _cache(**kw):
    """A cache struct whose pointers are aligned but lead nowhere: no call that is refused may follow them."""
    from llm_quant_b200 import _C
    f = dict(k_codes=4096, v_codes=4096, params=4096, positions=4096, mass=4096, state=4096, B=2, H=2, cap=4096, D=64)
    f.update(kw)
    return _C.KV4Cache(*[f[n] for n, _ in _C.KV4Cache._fields_])


def _form(**kw):
    from llm_quant_b200 import _C
    f = dict(Hq=4, Sq=1, q_sb=64, q_sh=64, q_ss=64, bound=4096, window=0, sm_scale=1.0, softcap=0.0, q_dtype=1, causal=0,
             accumulate=0)
    f.update(kw)
    return ctypes.byref(_C.KV4Attn(*[f[n] for n, _ in _C.KV4Attn._fields_]))


BAD = [({"D": 96}, "head dim"), ({"cap": 4040}, "multiple"), ({"B": 0}, "shape"), ({"H": -1}, "shape"),
       ({"cap": 1 << 31}, "too large"), ({"B": 1000, "H": 1000}, "too large"), ({"params": None}, "NULL"),
       ({"state": None}, "NULL"), ({"k_codes": 4097}, "aligned"), ({"params": 4104}, "aligned")]


@pytest.mark.parametrize("kw,word", BAD)
def test_bad_caches(lib, kw, word):
    c = ctypes.byref(_cache(**kw))
    calls = [lambda: lib.lq_kv4_append(c, 4096, 4096, 1, 1, 64, 64, 64, 64, 64, 64, None, None),
             lambda: lib.lq_kv4_dequant(c, 1, 1, 4096, 4096, None),
             lambda: lib.lq_kv4_evict(c, 4, 0, 0, 4096, 1 << 40, None),
             lambda: lib.lq_kv4_reset(c, None),
             lambda: lib.lq_kv4_attention(c, _form(), 4096, None, None, None, 4096, 4096, 1 << 40, None)]
    for call in calls:
        assert call() < 0
        assert word.encode() in lib.lq_last_error()
    assert lib.lq_kv4_attention_workspace_bytes(c, _form()) == 0


def test_bad_arguments(lib):
    c = ctypes.byref(_cache())

    def append(k=4096, v=4096, dt=1, S=1, st=(64,) * 6):
        return lib.lq_kv4_append(c, k, v, dt, S, *st, None, None)

    assert append(k=None) == -1 and append(dt=3) == -2 and append(S=-1) == -1
    assert append(k=4100) == -5 and append(st=(64, 64, 63, 64, 64, 64)) == -5
    assert append(S=0) == 0  # nothing to do
    assert lib.lq_kv4_dequant(c, 4097, 1, 4096, 4096, None) == -1
    assert lib.lq_kv4_dequant(c, 4, 3, 4096, 4096, None) == -2
    assert lib.lq_kv4_dequant(c, 4, 1, 4098, 4096, None) == -5
    assert lib.lq_kv4_dequant(c, 0, 1, None, None, None) == 0
    for keep, recent, sinks in ((0, 0, 0), (4, 5, 0), (4, 2, 3), (4, -1, 0)):
        assert lib.lq_kv4_evict(c, keep, recent, sinks, 4096, 1 << 40, None) == -1
    assert lib.lq_kv4_evict(c, 4096, 0, 0, None, 0, None) == 0  # nothing can be over it
    assert lib.lq_kv4_evict(c, 8, 0, 0, 4096, lib.lq_kv4_evict_workspace_bytes(2, 2, 4096, 8) - 1, None) == -1

    def attend(q=4096, out=4096, ws=4096, nbytes=1 << 40, **kw):
        return lib.lq_kv4_attention(c, _form(**kw), q, None, None, None, out, ws, nbytes, None)

    assert attend(Hq=3) == -1 and attend(Hq=0) == -1 and attend(q_dtype=3) == -2 and attend(softcap=-1.0) == -1
    assert attend(q=None) == -1 and attend(out=None) == -1 and attend(window=-1) == -1 and attend(window=1 << 31) == -1 and attend(Sq=-1) == -1
    assert attend(ws=None) == -1 and attend(ws=4100) == -5 and attend(q=4100) == -5 and attend(q_ss=66) == -5
    assert lib.lq_kv4_attention(c, None, 4096, None, None, None, 4096, 4096, 1 << 40, None) == -1
    need = lib.lq_kv4_attention_workspace_bytes(c, _form())
    assert need > 0 and attend(nbytes=need - 1) == -1
    assert attend(Sq=0) == 0


def test_caps_out_of_range(lib):
    c = ctypes.byref(_cache())
    for cap in (-1.0, 1e-21, 1e31, float("inf"), float("nan")):
        assert lib.lq_kv4_attention(c, _form(softcap=cap), 4096, None, None, None, 4096, 4096, 1 << 40, None) == -1
        assert b"softcap" in lib.lq_last_error()


def test_captures_are_looked_for_on_the_caches_device(monkeypatch):
    from llm_quant_b200 import packed_kv_cache as P
    now = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *exc):
            now[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)
    assert P._capturing(torch.device("cuda", 1)) and not P._capturing(torch.device("cuda", 0))
    st = object.__new__(P._LayerStore)
    st.device, st.B, st.cap, st.bound, st.captured = torch.device("cuda", 1), 1, 64, 5, False
    cache = L.PackedKVCache(1, 64)
    cache._layers[0] = st
    monkeypatch.setattr(cache, "_call", lambda *a: None)
    cache.reset()
    assert st.captured and cache.seq_len == 64 and now == [0]


def test_python_layer_without_a_gpu():
    with pytest.raises(ValueError):
        L.PackedKVCache(1, 0)
    with pytest.raises(ValueError):
        L.PackedKVCache(-1, 5)
    cache = L.PackedKVCache(2, 16)
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache.append(0, x, x)
    with pytest.raises(RuntimeError, match="empty"):
        cache.attend(1, x)
    with pytest.raises(IndexError):
        cache.get(2)
    assert cache.get(0) is None and cache.seq_len == 0
    cache.reset()
    cache.reset(1)
