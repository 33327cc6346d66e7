"""CPU-side checks of the adapter bank and of gradient clipping: what the classes
and the C entry points refuse before any launch (no GPU needed)."""

import ctypes

import pytest
import torch

import llm_quant_b200 as L


@pytest.fixture(scope="module")
def lib():
    from llm_quant_b200 import _C, build
    build.build()
    return _C.lib()


def _bank(**kw):
    """A bank whose pointers are aligned but lead nowhere: no call that is refused may follow them."""
    from llm_quant_b200 import _C
    f = dict(a=4096, b=4096, scaling=4096, L=4, R=16, K=64, N=128, dtype=2)
    f.update(kw)
    return ctypes.byref(_C.AdapterBank(*[f[n] for n, _ in _C.AdapterBank._fields_]))


def _form(n=4, x_stride=64, base_stride=0, out_stride=128, keep=0):
    from llm_quant_b200 import _C
    return ctypes.byref(_C.AdapterForm(n, x_stride, base_stride, out_stride, keep))


BAD = [({"a": None}, -1, "NULL"), ({"scaling": None}, -1, "NULL"), ({"dtype": 0}, -2, "fp16 or bf16"), ({"L": 0}, -6, "adapters"),
       ({"L": 8193}, -6, "adapters"), ({"R": 0}, -6, "rank"), ({"R": 129}, -6, "rank"), ({"K": 68}, -5, "multiples of 8"),
       ({"N": 4}, -6, "features"), ({"N": (1 << 22) + 8}, -6, "features"), ({"a": 4104}, -5, "aligned")]
HUGE = 1 << 40


@pytest.mark.parametrize("kw,status,word", BAD)
def test_bad_banks(lib, kw, status, word):
    b = _bank(**kw)
    for call in (lambda: lib.lq_adapter_forward(b, _form(), 4096, 4096, None, 4096, 4096, HUGE, None),
                 lambda: lib.lq_adapter_backward(b, _form(keep=1), 4096, 4096, 4096, 4096, HUGE, 4096, 4096, 4096, 2, 4096, HUGE, None)):
        assert call() == status
        assert word.encode() in lib.lq_last_error()


def test_bad_calls(lib):
    def forward(plan=4096, x=4096, base=None, out=4096, low=4096, nb=HUGE, **form):
        return lib.lq_adapter_forward(_bank(), _form(**form), plan, x, base, out, low, nb, None)

    assert forward(plan=None) == -1 and forward(plan=4104) == -1 and forward(n=-1) == -6 and forward(n=(1 << 24) + 1) == -6
    assert forward(x=None) == -5 and forward(x=4098) == -5 and forward(x_stride=68) == -5 and forward(x_stride=-64) == -1
    assert forward(out=None) == -5 and forward(out_stride=64) == -1 and forward(base=4104) == -5
    assert forward(base=4096, base_stride=136) == -1
    for kw in (dict(n=5000), dict(keep=1)):  # calls that leave something in low
        assert forward(low=None, **kw) == -1 and forward(low=4100, **kw) == -1 and forward(nb=64, **kw) == -1
    assert forward(n=0, plan=None, x=None, out=None, low=None, nb=0) == 0
    assert lib.lq_adapter_forward(_bank(), None, 4096, 4096, None, 4096, 4096, HUGE, None) == -1

    def backward(x=4096, dy=4096, ds=128, low=4096, nl=HUGE, dx=4096, da=4096, db=4096, dt=2, ws=4096, nb=HUGE, keep=1):
        return lib.lq_adapter_backward(_bank(), _form(out_stride=ds, keep=keep), 4096, x, dy, low, nl, dx, da, db, dt, ws, nb, None)

    assert backward(dt=1) == -2 and backward(dy=None) == -5 and backward(ds=100) == -5 and backward(low=None) == -1
    assert backward(x=None) == -5 and backward(dx=4104) == -5 and backward(ws=None) == -1 and backward(nb=8) == -1
    assert backward(nl=8) == -1 and backward(keep=0) == -1
    assert lib.lq_adapter_backward_workspace_bytes(None, 4) == 0 and lib.lq_adapter_backward_workspace_bytes(_bank(), -1) == 0
    assert lib.lq_adapter_low_bytes(None, _form()) == 0 and lib.lq_adapter_low_bytes(_bank(), None) == 0
    assert 0 < lib.lq_adapter_low_bytes(_bank(), _form(n=5000)) < lib.lq_adapter_low_bytes(_bank(), _form(n=5000, keep=1))


def test_bad_plans(lib):
    def plan(ids=4096, dt=5, n=4, seq=1, counts=None, num=4, p=4096):
        return lib.lq_adapter_plan(ids, dt, n, seq, counts, num, p, None)

    assert plan(dt=4) == -2 and plan(num=0) == -6 and plan(num=8193) == -6 and plan(n=-1) == -6 and plan(seq=1 << 23) == -6
    assert plan(ids=None) == -1 and plan(p=None) == -1 and plan(p=4100) == -1 and plan(n=0, ids=None, p=None) == 0
    assert lib.lq_adapter_plan_bytes(-1, 4) == 0 and lib.lq_adapter_plan_bytes(4, 0) == 0
    assert lib.lq_adapter_plan_bytes(1000, 4) >= 4 * (2000 + 12 + 4 * 12)


def test_bad_clips(lib):
    V, I64, I = ctypes.c_void_p * 2, ctypes.c_int64 * 2, ctypes.c_int * 2

    def clip(ptrs=(4096, 8192), out=None, n=(8, 8), dt=(0, 0), count=2, m=1.0, norm=4096, ws=4096, nb=1 << 40):
        return lib.lq_clip_grad_norm(V(*ptrs), None if out is None else V(*out), I64(*n), I(*dt), count, m, norm, ws, nb, None)

    assert clip(ptrs=(4096, None)) == -1 and clip(ptrs=(4098, 4096)) == -5 and clip(out=(4096, 4098)) == -5
    assert clip(n=(8, -1)) == -1 and clip(dt=(0, 3)) == -2 and clip(count=-1) == -1 and clip(m=-1.0) == -1
    assert clip(m=float("nan")) == -1 and clip(norm=None) == -1 and clip(ws=None) == -1 and clip(nb=8) == -1 and clip(ws=4100) == -1
    assert lib.lq_clip_workspace_bytes(-1) == 0


def test_refusals_without_a_device():
    for kw, word in (({"in_features": 65}, "in_features"), ({"out_features": 0}, "out_features"), ({"rank": 0}, "rank"),
                     ({"rank": 129}, "rank"), ({"num_adapters": 0}, "num_adapters"), ({"num_adapters": 8193}, "num_adapters")):
        args = dict(in_features=64, out_features=128, num_adapters=2, rank=8)
        args.update(kw)
        with pytest.raises(ValueError, match=word):
            L.AdapterBank(**args)
    with pytest.raises(TypeError):
        L.AdapterBank(64, 64, 2, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.AdapterBatch(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.GradClipper([torch.zeros(3)])
    with pytest.raises(ValueError, match="no layers"):
        L.AdapterBank.from_layers([])
    assert L.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3))], 1.0) == 0


def test_a_bank_of_layers():
    """Smaller ranks are filled up with zeros, lora_B is transposed."""
    layers = [L.QLoRALinear(64, 128, rank=r, alpha=2.0) for r in (4, 8)]
    for ql in layers:
        torch.nn.init.normal_(ql.lora_B)
    bank = L.AdapterBank.from_layers(layers, dtype=torch.float32)
    assert bank.rank == 8 and bank.scaling.tolist() == [0.5, 0.25]
    for i, ql in enumerate(layers):
        assert torch.equal(bank.lora_A[i, :ql.rank], ql.lora_A) and torch.equal(bank.lora_B[i, :ql.rank], ql.lora_B.t())
        assert not bank.lora_A[i, ql.rank:].any() and not bank.lora_B[i, ql.rank:].any()
    with pytest.raises(IndexError):
        bank.load_adapter(2, layers[0].lora_A, layers[0].lora_B, 1.0)
    with pytest.raises(ValueError):
        bank.load_adapter(0, layers[0].lora_A, layers[1].lora_B, 1.0)


def test_a_clipper_whose_memory_went(lib):
    """Addresses are taken once: a storage that was resized since is refused before any launch."""
    from llm_quant_b200 import _C
    for size in (0, 64, 1 << 20):
        g = torch.zeros(100)
        for clipper in (_C.ext().Clipper([torch.ones(8), g.detach()], None, []), _C.ext().Clipper([torch.ones(100)], [g.detach()], [])):
            kept = g.untyped_storage().size()
            g.untyped_storage().resize_(size)
            with pytest.raises(RuntimeError, match="storage of tensor . was resized"):
                clipper.clip(1.0)
            g.untyped_storage().resize_(kept)


class _Twice(torch.nn.Module):
    def forward(self, t):
        return 2 * t


def test_tensors_that_are_not_the_modules_parameters(lib):
    """Parametrized ones and those of a replica are found as attributes; no call
    fails before the device is asked for."""
    from types import SimpleNamespace
    batch = SimpleNamespace(_plan=torch.zeros(64, dtype=torch.uint8), tokens=4, num_adapters=2)
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    for change in ("parametrized", "replica"):
        bank = L.AdapterBank(64, 128, 2, 8)
        if change == "parametrized":
            torch.nn.utils.parametrize.register_parametrization(bank, "lora_A", _Twice())
        else:
            copy = bank._replicate_for_data_parallel()
            for name, t in (*bank._parameters.items(), *bank._buffers.items()):
                setattr(copy, name, t.detach())
            bank = copy
        with torch.no_grad():
            for call in (lambda: bank(x, batch), lambda: bank.add_(torch.zeros(4, 128, dtype=torch.bfloat16), x, batch)):
                with pytest.raises(RuntimeError, match="CUDA"):
                    call()
        if change == "parametrized":
            with pytest.raises(RuntimeError, match="computed"):
                bank.load_adapter(0, torch.zeros(8, 64), torch.zeros(128, 8), 1.0)


def test_forward_mode_is_refused(lib):
    """A tangent would be lost without a word."""
    import torch.autograd.forward_ad as fw
    from types import SimpleNamespace
    batch = SimpleNamespace(_plan=torch.zeros(64, dtype=torch.uint8), tokens=4, num_adapters=2)
    bank = L.AdapterBank(64, 128, 2, 8).requires_grad_(False)
    x, y = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 128, dtype=torch.bfloat16)
    with fw.dual_level():
        dual_x, dual_y = fw.make_dual(x, torch.ones_like(x)), fw.make_dual(y, torch.ones_like(y))
        for call in (lambda: bank(dual_x, batch), lambda: bank(x, batch, dual_y), lambda: bank.add_(dual_y, x, batch),
                     lambda: bank.add_(y, dual_x, batch)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="CUDA"):  # nothing has a tangent
            bank(x, batch, y)
        del bank.lora_B
        bank.lora_B = fw.make_dual(torch.zeros(2, 8, 128, dtype=torch.bfloat16), torch.ones(2, 8, 128, dtype=torch.bfloat16))
        with pytest.raises(RuntimeError, match="forward-mode"):
            bank(x, batch)


def test_first_calls_of_many_threads(lib, monkeypatch):
    """The bindings are loaded once, whoever comes first."""
    import importlib.machinery
    import threading
    import time
    from llm_quant_b200 import _C
    loads = []

    class Loader(importlib.machinery.ExtensionFileLoader):
        def create_module(self, spec):
            return None

        def exec_module(self, module):
            loads.append(module)
            time.sleep(0.2)

    monkeypatch.setattr(_C, "_ext", None)
    monkeypatch.setattr(importlib.machinery, "ExtensionFileLoader", Loader)
    got = []
    threads = [threading.Thread(target=lambda: got.append(_C.ext())) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(loads) == 1 and len(got) == 8 and all(m is loads[0] for m in got)


def test_build_without_torch_or_a_host_compiler(lib, tmp_path, monkeypatch, capfd):
    """The C library needs nvcc alone: it is linked whether or not its bindings can be."""
    import os
    import sys
    from llm_quant_b200 import build
    objects = {s: os.path.join(build.OBJDIR, s.replace(".cu", ".o")) for s in build._sources()}
    monkeypatch.setattr(build, "_compile", lambda src, force, verbose: objects[src])
    for name in ("LIBDIR", "OBJDIR", "LIB", "EXT"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    monkeypatch.setenv("CXX", str(tmp_path / "no_such_compiler"))
    with pytest.raises((OSError, RuntimeError)):
        build.build()
    assert os.path.exists(build.LIB) and not os.path.exists(build.EXT)
    os.remove(build.LIB)
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build() == build.LIB and os.path.exists(build.LIB) and not os.path.exists(build.EXT)
    assert "no torch" in capfd.readouterr().err


def test_bindings_are_built_for_one_torch(lib, monkeypatch):
    """Another torch: they are compiled again, and ones of another torch are not used."""
    import subprocess
    from llm_quant_b200 import _C, build
    ran = []

    def run(cmd, **kw):
        ran.append(cmd)
        return subprocess.CompletedProcess(cmd, 1, "", "stopped here")

    monkeypatch.setattr(build.subprocess, "run", run)
    build._compile_ext(False)
    assert not ran
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    with pytest.raises(RuntimeError, match="stopped here"):
        build._compile_ext(False)
    assert len(ran) == 1
    monkeypatch.setattr(_C, "_ext", None)
    with pytest.raises(RuntimeError, match="this is 1.0.0"):
        _C.ext()
