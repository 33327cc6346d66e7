"""llm_quant_b200.packed_kv_cache -- a KV cache held in 4 bits a value.

``QuantizedKVCache`` keeps a byte (or two) per code whatever the quantizer's
width, one length for the whole batch, and rebuilds nothing but plain
attention.  ``PackedKVCache`` stores two codes per byte (head dim 128: 136
bytes per token and head for K and V, of 512 in 16 bits), gives each sequence
of the batch a length of its own, attends single tokens and prompt chunks with
the score forms that models use (tanh cap, distance bias, sliding window,
prefix), collects the attention weight of each cached token, and evicts by it.

Quantization, per token and kv head over the head dim, in fp32:

    lo = min(0, min x)   hi = max(0, max x)   scale = bf16((hi - lo) / 15)
    zero = clamp(rint(-lo / scale), 0, 15)    code = clamp(rint(x / scale) + zero, 0, 15)
    value = (code - zero) * scale

This is KVCacheQuantizer(4, symmetric=False, PER_TOKEN) (kv_cache_quant.py:102-139,
168-193) but for three choices: the range always holds 0 (the reference clamps
a zero point that falls outside, and saturates), arithmetic is in fp32 whatever
the input's dtype (the reference rounds each operation to it, which turns an
all-zero fp16 token into NaN), and the scale is kept in bf16.

Lengths live on the device and nothing here reads them back, so every method
(but a layer's first ``append``, which makes its buffers, and ``check``) can be
captured into a CUDA graph and replayed: a replayed ``append`` goes on
where the last one stopped.  The host keeps an upper bound of them
(``seq_len``), which sizes what ``get``, ``positions`` and ``attention_mass``
return.  Once an ``append``, ``evict`` or ``reset`` was captured it is the
capacity for good, across ``reset`` too, since the host does not see replays;
an ``append`` that does not fit then no longer raises, its tokens are dropped
and counted (``dropped``).

One cache is used by one stream at a time (``attend`` without ``accumulate``
and ``get`` may overlap each other), as any tensor that is changed in place.
"""

from __future__ import annotations

import ctypes
import operator
from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import _C


class _LayerStore:
    """Device buffers of one layer."""

    def __init__(self, B: int, H: int, cap: int, D: int, device):
        self.B, self.H, self.cap, self.D, self.device = B, H, cap, D, device

        def new(fill, *shape, dtype=torch.int32):
            return torch.full(shape, fill, dtype=dtype, device=device)

        # codes are read in whole tiles, past the last token too: any code will do there
        self.k_codes = torch.empty(B, H, cap, D // 2, dtype=torch.uint8, device=device)
        self.v_codes = torch.empty_like(self.k_codes)
        self.params = torch.empty(B, H, cap, 2, dtype=torch.int32, device=device)
        self.positions = new(-1, B, H, cap)
        self.mass = new(0.0, B, H, cap, dtype=torch.float32)
        self.state = new(0, 2 * B + 4)
        self.bound = 0        # no sequence holds more tokens, as far as the host knows
        self.captured = False  # a change of the lengths was captured: its replays are not seen by the host
        self.emptied = False   # captured, and nothing but replays since the last reset
        self.c = _C.KV4Cache(self.k_codes.data_ptr(), self.v_codes.data_ptr(), self.params.data_ptr(),
                             self.positions.data_ptr(), self.mass.data_ptr(), self.state.data_ptr(),
                             B, H, cap, D)
        self.ref = ctypes.byref(self.c)
        self.forms: dict = {}  # attend's arguments as the entry point takes them

    def clear(self, capturing: bool) -> None:
        self.captured |= capturing
        self.bound = self.cap if self.captured else 0
        self.emptied = self.captured and not capturing


def _capturing(device: torch.device) -> bool:
    """Whether the stream that calls on `device` go to is being captured."""
    if device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device.index):
        return torch.cuda.is_current_stream_capturing()


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x with rows that the kernels can load: D contiguous, each row on a
    multiple of 4 elements.  A transposed projection qualifies as it is."""
    sb, sh, ss, sd = x.stride()
    if sd == 1 and not (sb | sh | ss) & 3 and x.data_ptr() % (4 * x.element_size()) == 0:
        return x
    return x.detach().clone(memory_format=torch.contiguous_format)


class PackedKVCache(nn.Module):
    """KV cache in 4 bits for inference (see the module's documentation).

    ``max_seq_len`` tokens of room for each sequence, rounded up to a multiple
    of 32 (the capacity, which replayed graphs may fill), are allocated per layer
    at its first chunk, whose shape [B, H, S, D] and device the cache keeps
    (head dim 64 or 128; float32, float16 or bfloat16 chunks).  That one cannot
    be captured into a graph; it may be empty (S = 0)."""

    def __init__(self, num_layers: int, max_seq_len: int):
        super().__init__()
        if num_layers < 0 or max_seq_len < 1:
            raise ValueError("PackedKVCache: num_layers must not be negative and max_seq_len at least 1")
        self.num_layers = num_layers
        self.max_seq_len = max_seq_len
        self._layers: list[Optional[_LayerStore]] = [None] * num_layers

    # -- helpers ---------------------------------------------------------------
    def _layer(self, layer_idx: int, what: str) -> _LayerStore:
        st = self._layers[layer_idx]
        if st is None:
            raise RuntimeError(f"PackedKVCache.{what}: layer {layer_idx} is empty")
        return st

    @staticmethod
    def _call(st: _LayerStore, name: str, *args) -> None:
        """Call an entry point on the layer's device and its current stream."""
        index = st.device.index
        if index == torch.cuda.current_device():
            _C.call(name, st.ref, *args, _C.raw_stream(index))
        else:
            with torch.cuda.device(index):
                _C.call(name, st.ref, *args, _C.raw_stream(index))

    @staticmethod
    def _vector(x, n: int, dtype, st: _LayerStore, what: str) -> int:
        if not isinstance(x, torch.Tensor) or x.dtype != dtype or x.shape != (n,) or x.device != st.device:
            raise ValueError(f"PackedKVCache.{what} must be a {dtype} tensor of {n} values on {st.device}")
        if not x.is_contiguous():
            raise ValueError(f"PackedKVCache.{what} must be contiguous")
        return x.data_ptr()

    # -- writing -----------------------------------------------------------------
    def append(self, layer_idx: int, key: torch.Tensor, value: torch.Tensor,
               counts: Optional[torch.Tensor] = None) -> None:
        """Quantize and store new K, V [B, H, S, D] behind what each sequence
        holds.  ``counts`` (int32 [B], on the device) says how many of the S
        tokens each sequence has, the rest being padding; default all.  Raises
        ValueError when S tokens might not fit into max_seq_len; what a replayed
        graph, or any call after a capture, appends past the capacity is dropped
        and counted (``dropped``)."""
        _C.require_cuda(key, value, what="PackedKVCache.append")
        _C.require_float(key, "PackedKVCache.append")
        if key.ndim != 4 or key.shape != value.shape:
            raise RuntimeError(f"PackedKVCache.append: key {list(key.shape)} and value {list(value.shape)} "
                               "must both be [B, H, S, D]")
        if key.dtype != value.dtype or key.device != value.device:
            raise TypeError("PackedKVCache.append: key and value must share dtype and device")
        B, H, S, D = key.shape
        st = self._layers[layer_idx]
        if st is None:
            if D not in (64, 128):
                raise ValueError(f"PackedKVCache: head dim {D}: 64 or 128 supported")
            if B == 0 or H == 0:
                raise ValueError("PackedKVCache: empty batch or no heads")
            if S > self.max_seq_len:
                raise ValueError(f"PackedKVCache.append: {S} tokens do not fit into {self.max_seq_len}")
            if B * H > 65535:
                raise ValueError("PackedKVCache: more than 65535 (sequence, head) pairs")
            if _capturing(key.device):
                # a captured allocation would be filled, and so the cache emptied, by every replay
                raise RuntimeError("PackedKVCache.append: a layer's first chunk (it may be empty, S = 0) must come "
                                   "before the capture")
            st = _LayerStore(B, H, (self.max_seq_len + 31) // 32 * 32, D, key.device)
            self._layers[layer_idx] = st
        elif (B, H, D) != (st.B, st.H, st.D) or key.device != st.device:
            raise RuntimeError(f"PackedKVCache.append: cache [{st.B}, {st.H}, *, {st.D}] on {st.device} vs new "
                               f"{list(key.shape)} on {key.device}")
        c = None if counts is None else self._vector(counts, B, torch.int32, st, "append: counts")
        if S == 0:
            return
        capturing = _capturing(st.device)
        if S > st.cap:
            raise ValueError(f"PackedKVCache.append: {S} tokens do not fit into {st.cap}")
        if not (capturing or st.captured) and st.bound + S > self.max_seq_len:
            raise ValueError(f"PackedKVCache.append: {S} more tokens than {st.bound} of {self.max_seq_len} "
                             "do not fit (evict, or reset)")
        k, v = _rows(key), _rows(value)
        ks, vs = k.stride(), v.stride()
        self._call(st, "lq_kv4_append", k.data_ptr(), v.data_ptr(), _C.TORCH_TO_LQ[k.dtype], S, ks[0], ks[1], ks[2],
                   vs[0], vs[1], vs[2], c)
        st.captured |= capturing
        st.bound = st.cap if st.captured else st.bound + S
        st.emptied = False

    def update(self, layer_idx: int, key: torch.Tensor, value: torch.Tensor,
               counts: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """``append``, then all cached K and V as values (``get``)."""
        self.append(layer_idx, key, value, counts)
        return self.get(layer_idx, dtype)

    # -- reading -----------------------------------------------------------------
    def get(self, layer_idx: int, dtype: torch.dtype = torch.float32) -> Optional[Tuple[torch.Tensor, torch.Tensor]]:
        """K, V [B, H, seq_len, D] as values in ``dtype``, zeros past a
        sequence's length, or None if the layer is empty."""
        st = self._layers[layer_idx]
        if st is None:
            return None
        if dtype not in _C.FLOAT_TYPES:
            raise TypeError(f"PackedKVCache.get: unsupported dtype {dtype} (float32, float16, bfloat16)")
        k = torch.empty(st.B, st.H, st.bound, st.D, dtype=dtype, device=st.device)
        v = torch.empty_like(k)
        if st.bound:
            self._call(st, "lq_kv4_dequant", st.bound, _C.TORCH_TO_LQ[dtype], k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, layer_idx: int, query: torch.Tensor, scale: Optional[float] = None, causal: bool = False, *,
               counts: Optional[torch.Tensor] = None, softcap: float = 0.0,
               slopes: Optional[torch.Tensor] = None, window: int = 0,
               prefix: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
        """softmax attention of query [B, Hq, Sq, D] over a layer's cached
        tokens, computed from the 4-bit codes; [B, Hq, Sq, D] in query's dtype.

        Hq is a multiple of the cached heads H (query head h reads kv head
        h // (Hq // H)).  The queries belong to the last tokens of their
        sequence: query i has position next - n + i, with n its sequence's
        ``counts`` (int32 [B]; default Sq) and ``next`` the position of the
        token that would be appended next.  Queries from n on are padding.
        For a query at position p and a token at position t,

            x = scale * q.k                      scale: default D ** -0.5
            x = softcap * tanh(x / softcap)      if softcap > 0
            x = x - slopes[h] * |p - t|          if slopes (float32 [Hq]) is given

        and the query sees the token if ((not causal or t <= p) and (window == 0
        or p - t < window)) or t < prefix[b] (int32 [B]).  A query that sees
        nothing gives zeros, and so does padding.  ``accumulate`` adds the
        weight that each token got from all queries to ``attention_mass``.

        Scores are summed in fp32 from exact products; with 16-bit queries each
        probability is rounded once, to fp16 beside the greatest of its row,
        before it meets the values.  Up to 16 such queries to a kv head also cut
        products below 2^-14 of a V scale times the probability (2^-10 at most for
        16 tokens); more round probabilities to 2^-24 of 2^7 and the greatest V
        scale among 128 slots: tokens with a scale below 2^-20 of that lose bits.
        Positions are int32, ``window`` is at most 2^30, a group has at most 4096
        query heads, ``softcap`` is 0 or 1e-20 to 1e30.

        Inference only: no gradient is computed."""
        st = self._layer(layer_idx, "attend")
        q = query if query.__class__ is torch.Tensor and query.ndim == 4 else self._query(st, query)
        # rounded up by 1/8 of an octave at most: the work is split by it, nothing else
        bound = st.cap if st.captured else st.bound
        step = 1 << max(5, bound.bit_length() - 4)
        bound = min((bound + step - 1) // step * step, st.cap)
        # numbers, whatever holds them: a tensor may hold another one at the next call
        softcap, window, causal, accumulate = float(softcap), operator.index(window), bool(causal), bool(accumulate)
        scale = st.D ** -0.5 if scale is None else float(scale)
        key = (q.dtype, q.shape, q.stride(), q.device, scale, causal, softcap, window, accumulate, bound)
        form = st.forms.get(key)
        if form is None or q.data_ptr() & 15:
            q = _rows(self._query(st, query))
            form = self._form(st, q, scale, causal, softcap, window, accumulate, bound)
            if q.data_ptr() == query.data_ptr():
                if len(st.forms) >= 256:
                    st.forms.clear()
                st.forms[key] = form
        ref, nbytes, _ = form
        B, Hq, Sq, D = q.shape
        cn = None if counts is None else self._vector(counts, B, torch.int32, st, "attend: counts")
        sl = None if slopes is None else self._vector(slopes, Hq, torch.float32, st, "attend: slopes")
        pf = None if prefix is None else self._vector(prefix, B, torch.int32, st, "attend: prefix")
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if Sq:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
            self._call(st, "lq_kv4_attention", ref, q.data_ptr(), cn, sl, pf, out.data_ptr(), _C.ptr(ws), nbytes)
        return out

    @staticmethod
    def _query(st: _LayerStore, query: torch.Tensor) -> torch.Tensor:
        _C.require_cuda(query, what="PackedKVCache.attend")
        _C.require_float(query, "PackedKVCache.attend")
        if query.ndim != 4 or query.shape[0] != st.B or query.shape[3] != st.D or query.shape[1] % st.H \
                or query.shape[1] == 0 or query.device != st.device:
            raise RuntimeError(f"PackedKVCache.attend: query {list(query.shape)} on {query.device} does not match "
                               f"the cache [{st.B}, {st.H}*G, *, {st.D}] on {st.device}")
        return query

    @staticmethod
    def _form(st: _LayerStore, q: torch.Tensor, scale: float, causal: bool, softcap: float, window: int,
              accumulate: bool, bound: int):
        """The call's arguments but for the tensors: checked once for each form."""
        if not (softcap == 0.0 or 1e-20 <= softcap <= 1e30):
            raise ValueError(f"PackedKVCache.attend: softcap {softcap} must be 0 (none) or 1e-20 to 1e30")
        if not 0 <= window <= 2 ** 30:
            raise ValueError(f"PackedKVCache.attend: window {window} must be 0 (none) to 2^30")
        sb, sh, ss, _ = q.stride()
        c = _C.KV4Attn(q.shape[1], q.shape[2], sb, sh, ss, bound, window, scale, softcap, _C.TORCH_TO_LQ[q.dtype],
                       causal, accumulate)
        return ctypes.byref(c), _C.lib().lq_kv4_attention_workspace_bytes(st.ref, ctypes.byref(c)), c

    # -- eviction ------------------------------------------------------------------
    def evict(self, layer_idx: int, keep: int, recent: int = 0, sinks: int = 0) -> None:
        """Cut every sequence back to ``keep`` tokens per kv head: the
        ``recent`` last ones and those at positions below ``sinks`` stay, then
        the ones with the greatest ``attention_mass`` (equal mass: from the
        lowest slot up; NaN counts as greatest, less than 0 as 0).  Heads keep tokens of their
        own.  Sequences that hold no more than ``keep`` are left alone."""
        st = self._layer(layer_idx, "evict")
        if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
            raise ValueError(f"PackedKVCache.evict: keep {keep} must be positive and hold the {recent} recent and "
                             f"{sinks} first tokens")
        capturing = _capturing(st.device)
        if keep >= st.cap or (keep >= st.bound and not st.captured and not capturing):
            return
        nbytes = _C.lib().lq_kv4_evict_workspace_bytes(st.B, st.H, st.cap, keep)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=st.device)
        self._call(st, "lq_kv4_evict", keep, recent, sinks, ws.data_ptr(), nbytes)
        if capturing:
            st.captured = True
            st.bound = st.cap
        elif not st.captured:
            st.bound = min(st.bound, keep)

    # -- what the cache holds --------------------------------------------------------
    def lengths(self, layer_idx: int) -> torch.Tensor:
        """Tokens that each sequence holds: int32 [B] on the device (the cache's own)."""
        st = self._layer(layer_idx, "lengths")
        return st.state[:st.B]

    def dropped(self, layer_idx: int) -> torch.Tensor:
        """Tokens that appends found no room for, replayed ones and those after
        a capture: int32 scalar on the device (the cache's own)."""
        st = self._layer(layer_idx, "dropped")
        return st.state[2 * st.B + 1]

    def check(self, layer_idx: int) -> None:
        """Wait for the layer's work and raise LQError if a kernel gave up a wait
        on the device (its results are incomplete then)."""
        st = self._layer(layer_idx, "check")
        status = int(st.state[2 * st.B + 3])
        if status:
            raise _C.LQError("PackedKVCache", status, "a wait on the device ran out")

    def positions(self, layer_idx: int) -> torch.Tensor:
        """Position of the token in each slot, -1 where it is empty: int32
        [B, H, seq_len] (the cache's own).  Until something is evicted slot t
        holds position t; then the order of slots means nothing."""
        st = self._layer(layer_idx, "positions")
        return st.positions.narrow(2, 0, st.bound)

    def attention_mass(self, layer_idx: int) -> torch.Tensor:
        """Attention weight that each slot's token collected (``attend`` with
        ``accumulate``), 0 where it is empty: float32 [B, H, seq_len], the
        cache's own, so it can be decayed or replaced in place."""
        st = self._layer(layer_idx, "attention_mass")
        return st.mass.narrow(2, 0, st.bound)

    def reset(self, layer_idx: Optional[int] = None) -> None:
        """Clear one layer, or all; the buffers stay, and so do captured graphs."""
        for st in self._layers if layer_idx is None else [self._layers[layer_idx]]:
            if st is not None:
                st.clear(_capturing(st.device))
                self._call(st, "lq_kv4_reset")

    @property
    def seq_len(self) -> int:
        """Tokens cached in layer 0: the most that any sequence may hold.  Only
        where a graph was captured and nothing but replays may have come since
        a ``reset`` does this wait for the device, to tell empty from not."""
        st = self._layers[0] if self.num_layers else None
        if st is None or st.emptied and not _capturing(st.device) and not st.state[:st.B].any():
            return 0
        return st.bound
