"""llm_quant_b200.adapters -- low-rank adapters of many requests beside one shared projection.

``QLoRALinear`` holds one adapter.  An ``AdapterBank`` holds L of them for a
projection from K to N features, an ``AdapterBatch`` says which of a batch's
tokens use which, and one call adds each token's own share to what the shared
projection gave:

    y_t = base_t + scaling[i] * lora_B[i]^T (lora_A[i] x_t)     i: the adapter of token t
    y_t = base_t                                                for a token without one

and, in training, gives the gradients of x, of all lora_A and of all lora_B.
The reference has no counterpart (its QLoRALinear.forward, qlora.py:306-312, is
the case of one adapter).

Activations are float16 or bfloat16.  Products are exact and summed in fp32,
``scaling * lora_A x`` is kept in fp32, and each output is rounded once.
Parameters may be float32 (a training run's master weights): they are rounded
to the activations' dtype at each call and their gradients come in float32.
Sums go in an order of their own: equal calls give equal bits.

Nothing here reads the device on the host, so plans, calls and their backward
passes can be captured into a CUDA graph and replayed (as for any module, with
no eager graph of the same parameters alive while a backward pass is captured).
"""

from __future__ import annotations

import ctypes
import math
from typing import Iterable, Optional

import torch
import torch.nn as nn

from . import _C

_HALF = (torch.float16, torch.bfloat16)
MAX_RANK, MAX_ADAPTERS, MAX_TOKENS = 128, 8192, 1 << 24


def _call(device: torch.device, name: str, *args) -> None:
    """Call an entry point on `device` and its current stream."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        _C.call(name, *args, _C.raw_stream(index))
    else:
        with torch.cuda.device(index):
            _C.call(name, *args, _C.raw_stream(index))


def _changed(t: torch.Tensor) -> None:
    """Tell autograd that a kernel wrote to t."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


class AdapterBatch:
    """Which tokens of a batch use which adapter: built once for all
    projections of a step, on the device.

    ``ids`` (int32 or int64 [n], on the device) is the adapter of each request;
    a value outside [0, num_adapters) (say -1) means none.  A request has
    ``seq_len`` tokens: the batch is n * seq_len tokens, as the rows of x
    [n, seq_len, K] or [n * seq_len, K].  ``counts`` (int32 [n], on the device)
    says how many of them are tokens, the rest being padding, which uses no
    adapter; default all.  ``ids`` of shape [n, seq_len] with ``seq_len`` left at
    1 give every token an adapter of its own.

    ``update`` writes the plan for new requests in place, so that a captured
    call sees them when it is replayed."""

    def __init__(self, ids: torch.Tensor, num_adapters: int, seq_len: int = 1,
                 counts: Optional[torch.Tensor] = None):
        _C.require_cuda(ids, what="AdapterBatch")
        if not 1 <= num_adapters <= MAX_ADAPTERS:
            raise ValueError(f"AdapterBatch: num_adapters {num_adapters} outside [1, {MAX_ADAPTERS}]")
        if seq_len < 0 or ids.numel() * seq_len > MAX_TOKENS:
            raise ValueError(f"AdapterBatch: {ids.numel()} requests of {seq_len} tokens outside [0, 2^24] tokens")
        self.num_adapters, self.seq_len, self.requests = num_adapters, seq_len, ids.numel()
        self.tokens = self.requests * seq_len
        self.device = ids.device
        self._sig = (self.tokens, num_adapters, ids.device)
        self._plan = torch.empty(_C.lib().lq_adapter_plan_bytes(self.tokens, num_adapters), dtype=torch.uint8,
                                 device=ids.device)
        self.update(ids, counts)

    def update(self, ids: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
        """The plan of other requests, as many and as long."""
        if ids.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"AdapterBatch: ids must be int32 or int64, not {ids.dtype}")
        if ids.device != self.device or ids.numel() != self.requests:
            raise ValueError(f"AdapterBatch: {ids.numel()} ids on {ids.device}, expected {self.requests} on {self.device}")
        if counts is not None and (counts.dtype != torch.int32 or counts.device != self.device
                                   or counts.numel() != self.requests):
            raise ValueError(f"AdapterBatch: counts must be {self.requests} int32 values on {self.device}")
        if self.tokens == 0:
            return
        ids = ids.contiguous()
        counts = None if counts is None else counts.contiguous()
        _changed(self._plan)  # a backward pass of the old plan raises
        _call(self.device, "lq_adapter_plan", ids.data_ptr(), _C.dt(ids), self.requests, self.seq_len, _C.ptr(counts),
              self.num_adapters, self._plan.data_ptr())

    def check(self) -> None:
        """Wait for the batch's work and raise LQError if a kernel gave up a
        wait on the device since the last ``update`` (its results are
        incomplete then)."""
        status = int(self._plan[:4].view(torch.int32)) if self.tokens else _C.OK
        if status:
            raise _C.LQError("AdapterBatch", status, "a wait on the device ran out")


def _row_stride(x: torch.Tensor) -> Optional[int]:
    """Elements from row to row of x [..., width], or None where the kernels
    cannot read its rows as they lie: side by side values, one stride over all
    leading dimensions, rows on 16 bytes."""
    width = x.shape[-1]
    if x.numel() <= width or x.is_contiguous():
        return width if x.numel() == 0 or x.stride(-1) == 1 else None
    if x.stride(-1) != 1:
        return None
    rows, stride = 1, None
    for n, st in zip(reversed(x.shape[:-1]), reversed(x.stride()[:-1])):
        if n == 1:
            continue
        if stride is None:
            stride = st
        elif st != rows * stride:
            return None
        rows *= n
    return stride if stride >= 0 and stride % 8 == 0 else None


class AdapterBank(nn.Module):
    """L adapters of one projection (see the module's documentation).

    ``lora_A`` [L, rank, in_features], ``lora_B`` [L, rank, out_features] (each
    adapter's lora_B of QLoRALinear transposed; zeros at the start) and
    ``scaling`` [L] (float32; alpha / rank).  in_features and out_features are
    multiples of 8, rank is at most 128: a smaller adapter's rows are filled
    up with zeros and stay so in training."""

    def __init__(self, in_features: int, out_features: int, num_adapters: int, rank: int = 16, alpha: float = 16.0,
                 *, dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        for name, n in (("in_features", in_features), ("out_features", out_features)):
            if n < 8 or n % 8 or n > 1 << 22:
                raise ValueError(f"AdapterBank: {name} {n} must be a multiple of 8 up to 2^22")
        if not 1 <= rank <= MAX_RANK:
            raise ValueError(f"AdapterBank: rank {rank} outside [1, {MAX_RANK}]")
        if not 1 <= num_adapters <= MAX_ADAPTERS:
            raise ValueError(f"AdapterBank: num_adapters {num_adapters} outside [1, {MAX_ADAPTERS}]")
        if dtype not in _C.FLOAT_TYPES:
            raise TypeError(f"AdapterBank: unsupported dtype {dtype} (float32, float16, bfloat16)")
        self.in_features, self.out_features = in_features, out_features
        self.num_adapters, self.rank = num_adapters, rank
        self.lora_A = nn.Parameter(torch.empty(num_adapters, rank, in_features, dtype=dtype, device=device))
        self.lora_B = nn.Parameter(torch.zeros(num_adapters, rank, out_features, dtype=dtype, device=device))
        self.register_buffer("scaling", torch.full((num_adapters,), alpha / rank, dtype=torch.float32, device=device))
        bound = 1.0 / math.sqrt(in_features)  # as QLoRALinear's
        nn.init.uniform_(self.lora_A, -bound, bound)
        self._c = (None, None)  # the bank's addresses, and the bank as the entry points take it
        self._shapes = (self.lora_A.shape, self.lora_B.shape)
        self._forms: dict = {}  # calls' shapes and strides as the entry points take them

    @classmethod
    def from_layers(cls, layers: Iterable, *, dtype: torch.dtype = torch.bfloat16) -> "AdapterBank":
        """The adapters of several QLoRALinear of one shape, as one bank."""
        layers = list(layers)
        if not layers:
            raise ValueError("AdapterBank.from_layers: no layers")
        bank = cls(layers[0].in_features, layers[0].out_features, len(layers), max(ql.rank for ql in layers),
                   dtype=dtype, device=layers[0].lora_A.device)
        for i, ql in enumerate(layers):
            bank.load_adapter(i, ql.lora_A, ql.lora_B, ql.scaling)
        return bank

    @torch.no_grad()
    def load_adapter(self, index: int, lora_A: torch.Tensor, lora_B: torch.Tensor, scaling: float) -> None:
        """Adapter `index` from lora_A [r, in_features] and lora_B
        [out_features, r], r up to the bank's rank."""
        r = lora_A.shape[0]
        if not 0 <= index < self.num_adapters:
            raise IndexError(f"AdapterBank.load_adapter: {index} outside [0, {self.num_adapters})")
        if lora_A.shape != (r, self.in_features) or lora_B.shape != (self.out_features, r) or r > self.rank:
            raise ValueError(f"AdapterBank.load_adapter: lora_A {list(lora_A.shape)} and lora_B {list(lora_B.shape)} for "
                             f"a bank of {self.in_features} to {self.out_features} features, rank {self.rank}")
        self.lora_A[index, :r] = lora_A
        self.lora_A[index, r:] = 0
        self.lora_B[index, :r] = lora_B.t()
        self.lora_B[index, r:] = 0
        self.scaling[index] = scaling

    # -- calls -------------------------------------------------------------------
    def _weights(self, x: torch.Tensor):
        """(the bank as the entry points take it, by reference, and the tensors
        that it points to: lora_A, lora_B in x's dtype, scaling)"""
        p = self._parameters
        a, b, s = p["lora_A"], p["lora_B"], self._buffers["scaling"]
        key = (a.data_ptr(), b.data_ptr(), s.data_ptr(), a.dtype, a.numel(), b.numel(), a.is_contiguous(), x.dtype, x.device)
        known, ref = self._c
        if known == key:
            return ref, a, b, s
        dev = x.device
        if a.device != dev or b.device != dev or s.device != dev:
            raise RuntimeError(f"AdapterBank: x on {dev}, the bank on {a.device}")
        if a.dtype != b.dtype or s.dtype != torch.float32:
            raise TypeError(f"AdapterBank: lora_A is {a.dtype}, lora_B {b.dtype}, scaling {s.dtype} (expected float32)")
        if a.shape != self._shapes[0] or b.shape != self._shapes[1] or s.numel() != self.num_adapters:
            raise RuntimeError(f"AdapterBank: lora_A {list(a.shape)}, lora_B {list(b.shape)} are not the bank's")
        as_is = a.dtype == x.dtype
        if not as_is:
            a, b = a.detach().to(x.dtype), b.detach().to(x.dtype)
        if not (a.is_contiguous() and b.is_contiguous() and s.is_contiguous()) or (a.data_ptr() | b.data_ptr()) & 15:
            a, b, s = (t.detach().clone(memory_format=torch.contiguous_format) for t in (a, b, s))
            as_is = False
        ref = self._struct(a, b, s)
        if as_is:
            self._c = (key, ref)  # the struct itself is never changed
        return ref, a, b, s

    def _struct(self, a: torch.Tensor, b: torch.Tensor, s: torch.Tensor):
        return ctypes.byref(_C.AdapterBank(a.data_ptr(), b.data_ptr(), s.data_ptr(), self.num_adapters, self.rank,
                                           self.in_features, self.out_features, _C.dt(a)))

    def _form(self, key, x: torch.Tensor, batch: AdapterBatch, base: Optional[torch.Tensor], keep: bool,
              inplace: bool):
        """What a call's shapes and strides come to, checked once for each such
        form: (form, bytes of `low`, shape of the result, whether x / base are to be
        laid out first, form struct)."""
        _C.require_cuda(x, what="AdapterBank")
        if x.dtype not in _HALF:
            raise TypeError(f"AdapterBank: unsupported dtype {x.dtype} (float16, bfloat16)")
        if x.shape[-1:] != (self.in_features,) or x.numel() != batch.tokens * self.in_features:
            raise RuntimeError(f"AdapterBank: x {list(x.shape)} is not {batch.tokens} tokens of {self.in_features} features")
        if batch.num_adapters != self.num_adapters:
            raise ValueError(f"AdapterBank: a batch for {batch.num_adapters} adapters, a bank of {self.num_adapters}")
        if batch.device != x.device:
            raise RuntimeError(f"AdapterBank: x on {x.device}, the batch on {batch.device}")
        shape = x.shape[:-1] + (self.out_features,)
        if base is not None and (base.dtype != x.dtype or base.device != x.device or base.shape != shape):
            raise RuntimeError(f"AdapterBank: base {list(base.shape)} {base.dtype} on {base.device} for x {list(x.shape)} "
                               f"{x.dtype} on {x.device}")
        xs = _row_stride(x)
        bs = 0 if base is None else _row_stride(base)
        if inplace and (bs is None or batch.tokens > 1 and bs < self.out_features):
            raise ValueError(f"AdapterBank.add_: y {list(base.shape)} with strides {list(base.stride())} must be rows on 16 bytes")
        c = _C.AdapterForm(batch.tokens, self.in_features if xs is None else xs, self.out_features if bs is None else bs,
                           bs if inplace else self.out_features, keep)
        ref = ctypes.byref(c)
        bank = _C.AdapterBank(None, None, None, self.num_adapters, self.rank, self.in_features, self.out_features, _C.dt(x))
        low = _C.lib().lq_adapter_low_bytes(ctypes.byref(bank), ref)
        form = (ref, low, shape, xs is None, bs is None, c)
        if len(self._forms) >= 256:
            self._forms.clear()
        self._forms[key] = form
        return form

    def _run(self, x: torch.Tensor, batch: AdapterBatch, base: Optional[torch.Tensor], keep: bool, inplace: bool):
        """(out, low, form, bank by reference, a, b, scaling, x as it was read)"""
        if base is None:
            key = (x.dtype, x.shape, x.stride(), x.device, batch._sig, keep)
        else:
            key = (x.dtype, x.shape, x.stride(), x.device, batch._sig, keep, inplace, base.dtype, base.shape, base.stride(),
                   base.device)
        form = self._forms.get(key)
        if form is None:
            form = self._form(key, x, batch, base, keep, inplace)
        ref, nbytes, shape, copy_x, copy_base, _ = form
        bank, a, b, s = self._weights(x)
        dev = x.device
        if copy_x:
            x = x.contiguous() if not x.is_contiguous() else x.clone()
        at = x.data_ptr()
        if at & 15:
            if not copy_x and not x.is_contiguous():  # the form's strides are x's
                return self._run(x.contiguous(), batch, base, keep, inplace)
            x = x.clone()
            at = x.data_ptr()
        base_at = None
        if base is not None:
            if copy_base:
                base = base.contiguous() if not base.is_contiguous() else base.clone()
            base_at = base.data_ptr()
            if base_at & 15:
                if inplace:
                    raise ValueError("AdapterBank.add_: y must be rows on 16 bytes")
                return self._run(x, batch, base.clone(memory_format=torch.contiguous_format), keep, inplace)
        out = base if inplace else torch.empty(shape, dtype=x.dtype, device=dev)
        low = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        if batch.tokens:
            _call(dev, "lq_adapter_forward", bank, ref, batch._plan.data_ptr(), at, base_at,
                  out.data_ptr(), None if low is None else low.data_ptr(), nbytes)
        return out, low, form, bank, a, b, s, x

    def forward(self, x: torch.Tensor, batch: AdapterBatch, base: Optional[torch.Tensor] = None) -> torch.Tensor:
        """base [..., out_features] (default zeros) plus each token's adapter of
        x [..., in_features], whose leading dimensions are the batch's tokens."""
        if torch.is_grad_enabled():
            p = self._parameters
            a, b = p["lora_A"], p["lora_B"]
            if x.requires_grad or a.requires_grad or b.requires_grad or base is not None and base.requires_grad:
                return _Adapters.apply(x, a, b, base, self, batch)
        return self._run(x, batch, base, False, False)[0]

    def add_(self, y: torch.Tensor, x: torch.Tensor, batch: AdapterBatch) -> torch.Tensor:
        """y += each token's adapter of x, in place; no gradient (call it under
        ``torch.no_grad()``).  Rows of tokens without an adapter are not written."""
        if torch.is_grad_enabled() and (x.requires_grad or y.requires_grad or self.lora_A.requires_grad
                                        or self.lora_B.requires_grad):
            raise RuntimeError("AdapterBank.add_: no gradient is computed here (use forward, or torch.no_grad())")
        self._run(x, batch, y, False, True)
        _changed(y)
        return y

    def extra_repr(self) -> str:
        return (f"in={self.in_features}, out={self.out_features}, adapters={self.num_adapters}, rank={self.rank}, "
                f"dtype={self.lora_A.dtype}")


class _Adapters(torch.autograd.Function):
    """AdapterBank.forward with the gradients of x, lora_A, lora_B and base."""

    @staticmethod
    def forward(ctx, x, lora_A, lora_B, base, bank, batch):
        y, low, form, ref, a, b, s, rows = bank._run(x, batch, base, True, False)
        ctx.save_for_backward(rows, a, b)  # the weights as the call rounded them
        # low is nobody else's; scaling and the plan may be written to
        ctx.call = (low, form, ref, s, s._version, batch._plan, batch._plan._version, x.shape, lora_A.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():
            raise RuntimeError("AdapterBank: gradients of gradients are not computed")
        want_x, want_a, want_b, want_base = ctx.needs_input_grad[:4]
        dx = da = db = None
        if want_x or want_a or want_b:
            x, a, b = ctx.saved_tensors
            low, (form, nbytes, _, _, _, c), ref, s, s_version, plan, plan_version, shape, dtype = ctx.call
            if s._version != s_version or plan._version != plan_version:
                raise RuntimeError("AdapterBank: scaling or the batch's plan has been modified by an inplace operation "
                                   "since the forward pass")
            dev = x.device
            if want_x:
                dx = torch.empty(shape, dtype=x.dtype, device=dev)
            if want_a:
                da = torch.empty(a.shape, dtype=dtype, device=dev)
            if want_b:
                db = torch.empty(b.shape, dtype=dtype, device=dev)
            out_features = b.shape[2]
            d = dy
            stride = out_features
            if not d.is_contiguous():
                stride = _row_stride(d)
            if stride is None or d.data_ptr() & 15:
                d = d.clone(memory_format=torch.contiguous_format)
                stride = out_features
            if stride != c.out_stride:
                form = ctypes.byref(_C.AdapterForm(c.n, c.x_stride, 0, stride, 1))
            ws_bytes = _C.lib().lq_adapter_backward_workspace_bytes(ref, c.n)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            _call(dev, "lq_adapter_backward", ref, form, plan.data_ptr(), x.data_ptr(), d.data_ptr(),
                  None if low is None else low.data_ptr(), nbytes, None if dx is None else dx.data_ptr(),
                  None if da is None else da.data_ptr(), None if db is None else db.data_ptr(), _C.TORCH_TO_LQ[dtype],
                  ws.data_ptr(), ws_bytes)
        return dx, da, db, dy if want_base else None, None, None
