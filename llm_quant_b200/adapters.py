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

Activations are float16 or bfloat16.  Products are exact and summed in fp32;
``scaling * lora_A x`` meets lora_B in fp32 or as two 16-bit parts (off by 2^-16
of itself in bfloat16; in float16 2^-22, or 2^-37 of the greatest value beside it
if that is more: of its token's or, in the sums of lora_A's and lora_B's gradients,
of its adapter's), and each output is rounded once.
Parameters may be float32 (a training run's master weights): they are rounded
to the activations' dtype at each call and their gradients come in float32.
Sums go in an order of their own: equal calls give equal bits.  An infinite x or
gradient gives what the formulas give; an infinite weight may give NaN where they
give an infinity.

Nothing here reads the device on the host, so plans, calls and their backward
passes can be captured into a CUDA graph and replayed (as for any module, with
no eager graph of the same parameters alive while a backward pass is captured).
"""

from __future__ import annotations

import math
from typing import Iterable, Optional

import torch
import torch.nn as nn

from . import _C

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
        """Wait for the device, whichever streams the batch's work went to, and
        raise LQError if a kernel gave up a wait there since the last ``update``
        (its results are incomplete then)."""
        torch.cuda.synchronize(self.device)
        status = int(self._plan[:4].view(torch.int32)) if self.tokens else _C.OK
        if status:
            raise _C.LQError("AdapterBatch", status, "a wait on the device ran out")


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

    def _apply(self, fn, recurse=True):
        """``scaling`` goes where the parameters go, and stays float32."""
        scaling = self.scaling
        super()._apply(fn, recurse)
        if self.scaling.dtype != torch.float32:
            self.scaling = scaling.to(self.scaling.device)
        return self

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
        if nn.utils.parametrize.is_parametrized(self):
            raise RuntimeError("AdapterBank.load_adapter: the bank's tensors are computed (nn.utils.parametrize)")
        if lora_A.shape != (r, self.in_features) or lora_B.shape != (self.out_features, r) or r > self.rank:
            raise ValueError(f"AdapterBank.load_adapter: lora_A {list(lora_A.shape)} and lora_B {list(lora_B.shape)} for "
                             f"a bank of {self.in_features} to {self.out_features} features, rank {self.rank}")
        self.lora_A[index, :r] = lora_A
        self.lora_A[index, r:] = 0
        self.lora_B[index, :r] = lora_B.t()
        self.lora_B[index, r:] = 0
        self.scaling[index] = scaling

    def _tensors(self):
        """lora_A, lora_B and scaling: from the module's own tables (0.2 us less of a
        call), and as attributes where they are not in these, as of a parametrized
        bank or a replica."""
        p = self._parameters
        try:
            return p["lora_A"], p["lora_B"], self._buffers["scaling"]
        except KeyError:
            return self.lora_A, self.lora_B, self.scaling

    # -- calls (checked, allocated for and differentiated in csrc/lq_torch.cpp) ------
    def forward(self, x: torch.Tensor, batch: AdapterBatch, base: Optional[torch.Tensor] = None) -> torch.Tensor:
        """base [..., out_features] (default zeros) plus each token's adapter of
        x [..., in_features], whose leading dimensions are the batch's tokens."""
        return _C.ext().adapters_forward(x, *self._tensors(), base, batch._plan, batch.tokens, batch.num_adapters)

    def add_(self, y: torch.Tensor, x: torch.Tensor, batch: AdapterBatch) -> torch.Tensor:
        """y += each token's adapter of x, in place; no gradient (call it under
        ``torch.no_grad()``).  Rows of tokens without an adapter are not written.  y
        may be x, or share x's buffer, where no row of y overlaps another token's
        row of x."""
        _C.ext().adapters_add_(y, x, *self._tensors(), batch._plan, batch.tokens, batch.num_adapters)
        return y

    def extra_repr(self) -> str:
        return (f"in={self.in_features}, out={self.out_features}, adapters={self.num_adapters}, rank={self.rank}, "
                f"dtype={self.lora_A.dtype}")
