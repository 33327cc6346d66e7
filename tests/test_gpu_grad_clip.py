"""GPU tests of GradClipper and clip_grad_norm_ against the formula in 64 bits.

Tolerances.  The squares of 8 neighbours are summed in fp32 (8 roundings of
2^-24 of a sum of non-negative terms), everything else in fp64, and the root
halves a relative error: the norm is off by 4 * 2^-24 + 2^-24 (its own rounding)
of itself at most.  The factor is rounded to fp32, and so is its product with a
value before it is rounded to the value's type: half a step of that type and
2 * 2^-24 + 4 * 2^-24 of the result."""

import math

import pytest
import torch

import llm_quant_b200 as L

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def expected(grads, max_norm):
    norm = math.sqrt(math.fsum(float(g.double().square().sum()) for g in grads))
    c = min(1.0, max_norm / (norm + 1e-6))
    return norm, [g.double() * c for g in grads]


def check(got_norm, got, grads, max_norm):
    norm, want = expected(grads, max_norm)
    assert abs(float(got_norm) - norm) <= 5 * 2.0 ** -24 * norm
    for g, w in zip(got, want):
        half = torch.finfo(g.dtype).eps / 2
        tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[g.dtype]
        assert bool(((g.double() - w).abs() <= (half + 6 * 2.0 ** -24) * w.abs() + tiny).all())


def rand(n, dt, seed=0, scale=1.0):
    return (torch.randn(n, generator=torch.Generator(DEV).manual_seed(seed), device=DEV) * scale).to(dt)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("sizes", [[1], [2, 3, 5], [16384], [16383, 16385], [1000003], [7] * 40, [513, 0, 100001, 1, 8, 65536],
                                   [3] * 300, [100] * 2500])
def test_sizes(sizes, dt):
    grads = [rand(n, TYPES[dt], i) for i, n in enumerate(sizes)]
    total = expected(grads, 1.0)[0]
    for max_norm in (total / 3, total * 3, 0.0):
        work = [g.clone() for g in grads]
        norm = L.GradClipper(work).clip(max_norm)
        assert norm.shape == () and norm.dtype == torch.float32
        check(norm, work, grads, max_norm)
        if max_norm > total:
            assert all(torch.equal(a, b) for a, b in zip(work, grads))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("n", [1, 7, 40, 8191, 70001])
def test_every_address(dt, n):
    """Sources and results off 16 bytes in every way that the type allows; their neighbours stay."""
    t = TYPES[dt]
    step = 16 // torch.finfo(t).bits * 8
    for a in range(step):
        for b in {0, 1, (a + 1) % step, step - 1}:
            src, dst = rand(n + 2 * step, t, a), rand(n + 2 * step, t, 99)
            g, o = src[a:a + n], dst[b:b + n]
            kept = dst.clone()
            norm = L.GradClipper([g], [o]).clip(0.5)
            check(norm, [o], [g], 0.5)
            assert torch.equal(dst[:b], kept[:b]) and torch.equal(dst[b + n:], kept[b + n:])
            inplace = src.clone()
            L.GradClipper([inplace[a:a + n]]).clip(0.5)
            assert torch.equal(inplace[a:a + n], o)
            assert torch.equal(inplace[:a], src[:a]) and torch.equal(inplace[a + n:], src[a + n:])


def test_mixed_types_and_parts_of_a_buffer():
    sizes = [5000, 77, 33333, 2, 12345]
    grads = [rand(n, t, n) for n, t in zip(sizes, [torch.float32, torch.bfloat16, torch.float16, torch.float32, torch.bfloat16])]
    check(L.GradClipper(work := [g.clone() for g in grads]).clip(1.5), work, grads, 1.5)
    grads = [rand(n, torch.bfloat16, n) for n in sizes]
    flat = torch.zeros(sum(sizes), dtype=torch.bfloat16, device=DEV)
    kept = [g.clone() for g in grads]
    check(L.GradClipper(grads, list(flat.split(sizes))).clip(2.0), list(flat.split(sizes)), grads, 2.0)
    assert all(torch.equal(a, b) for a, b in zip(grads, kept))


def test_large():
    grads = [rand(40_000_003, torch.bfloat16, 1, 0.01), rand(30_000_001, torch.float32, 2, 0.01)]
    work = [g.clone() for g in grads]
    first = L.GradClipper(work).clip(1.0)
    check(first, work, grads, 1.0)
    again = [g.clone() for g in grads]
    assert torch.equal(L.GradClipper(again).clip(1.0), first)  # equal calls, equal bits
    assert all(torch.equal(a, b) for a, b in zip(work, again))


@pytest.mark.parametrize("dt,scale", [("fp32", 1e30), ("fp32", 1e-30), ("bf16", 1e30), ("bf16", 1e-35), ("fp16", 60000.0),
                                      ("fp16", 1e-6)])
def test_range_of_values(dt, scale):
    """Squares that fp32 cannot hold."""
    g = (torch.rand(5003, device=DEV, generator=torch.Generator(DEV).manual_seed(3)) * scale).to(TYPES[dt])
    g[100:3000] = 0
    norm, _ = expected([g], 1.0)
    for max_norm in (norm / 2, norm * 4):
        work = g.clone()
        got = L.GradClipper([work]).clip(max_norm)
        check(got, [work], [g], max_norm)


def test_not_finite():
    for dt in TYPES.values():
        g = rand(3000, dt)
        g[5] = float("inf")
        work = g.clone()
        assert float(L.GradClipper([work]).clip(1.0)) == float("inf")
        assert work[5].isnan() and not torch.cat([work[:5], work[6:]]).any()
        g[2000] = float("nan")
        other = rand(10, dt)
        norm = L.GradClipper([g, other]).clip(1.0)
        assert norm.isnan() and g.isnan().all() and other.isnan().all()


def test_zeros_and_no_limit():
    g = torch.zeros(5000, dtype=torch.bfloat16, device=DEV)
    assert float(L.GradClipper([g]).clip(1.0)) == 0 and not g.any()
    g = rand(5000, torch.float32)
    kept = g.clone()
    assert abs(float(L.GradClipper([g]).clip(float("inf"))) - float(kept.double().norm())) < 1e-4
    assert torch.equal(g, kept)


def test_shapes_and_parameters():
    p = [torch.nn.Parameter(rand(600, torch.float32, i).view(20, 30)) for i in range(4)]
    for i, q in enumerate(p[:3]):
        q.grad = rand(600, torch.float32, 10 + i).view(20, 30) if i else rand(600, torch.float32).view(30, 20).t()
    grads = [q.grad.clone() for q in p[:3]]
    ref = [torch.nn.Parameter(q.detach().clone()) for q in p]
    for q, r in zip(p, ref):
        r.grad = None if q.grad is None else q.grad.clone()
    norm = L.clip_grad_norm_(iter(p), 3.0)
    check(norm, [q.grad for q in p[:3]], grads, 3.0)
    theirs = torch.nn.utils.clip_grad_norm_(ref, 3.0)
    assert abs(float(theirs) - float(norm)) <= 1e-5 * float(norm)
    assert float(L.clip_grad_norm_([torch.nn.Parameter(rand(3, torch.float32))], 1.0)) == 0
    assert float(L.clip_grad_norm_(p[1], 1e9)) > 0


def test_refusals():
    g = rand(100, torch.float32)
    with pytest.raises(ValueError, match="no tensors"):
        L.GradClipper([])
    with pytest.raises(ValueError, match="overlaps"):
        L.GradClipper([g, g])
    with pytest.raises(ValueError, match="overlaps"):
        L.GradClipper([g[:60], g[50:]])
    with pytest.raises(ValueError, match="overlaps"):
        L.GradClipper([g[:50], rand(50, torch.float32)], [g[40:90], rand(50, torch.float32)])
    with pytest.raises(ValueError, match="overlaps"):
        L.GradClipper([g[:50], g[50:]], [rand(100, torch.float32)[:50], g[:50]])
    with pytest.raises(ValueError, match="out"):
        L.GradClipper([g], [])
    with pytest.raises(ValueError, match="shape, dtype"):
        L.GradClipper([g], [g.half()])
    with pytest.raises(ValueError, match="side by side"):
        L.GradClipper([g[::2]])
    with pytest.raises(TypeError):
        L.GradClipper([g.double()])
    with pytest.raises(RuntimeError, match="CUDA"):
        L.GradClipper([g.cpu()])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            L.GradClipper([g]).clip(bad)


def test_captured_and_streams():
    g = [rand(50001, torch.bfloat16, i) for i in range(5)]
    src = [t.clone() for t in g]
    clipper = L.GradClipper(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clipper.clip(1.0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clipper.clip(1.0)
    for k in (1.0, 5.0):
        for t, s in zip(g, src):
            t.copy_(s * k)
        before = [t.clone() for t in g]
        graph.replay()
        check(norm, g, before, 1.0)


def test_memory_stays():
    """A tensor that is given other memory leaves the clipper's as it was."""
    g = rand(1000, torch.float32)
    kept = g.detach()
    clipper = L.GradClipper([g])
    g.data = rand(10, torch.float32)
    before = kept.clone()
    check(clipper.clip(0.5), [kept], [before], 0.5)


def test_versions():
    """A graph that saved a clipped tensor raises; parts of one buffer count as the buffer."""
    x = rand(100, torch.float32).requires_grad_(True)
    g = rand(100, torch.float32)
    y = (x * g).sum()
    L.GradClipper([g]).clip(0.5)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    flat = rand(300, torch.bfloat16)
    before = flat._version
    L.GradClipper(list(flat.split(100))).clip(0.5)
    assert flat._version == before + 1
    with torch.inference_mode():
        h = rand(50, torch.float32)
        check(L.GradClipper([h]).clip(0.5), [h], [rand(50, torch.float32)], 0.5)


def test_offsets_over_32_bits():
    """More than 2^31 values in a tensor, its result off 16 bytes."""
    n = 2 ** 31 + 12345
    g = torch.empty(n, dtype=torch.bfloat16, device=DEV)
    step = 1 << 27
    for i in range(0, n, step):
        g[i:i + step].normal_(std=0.01, generator=torch.Generator(DEV).manual_seed(i))
    out = torch.empty(n + 8, dtype=torch.bfloat16, device=DEV)[3:n + 3]
    norm = L.GradClipper([g], [out]).clip(1.0)
    total = math.sqrt(math.fsum(float(g[i:i + step].double().square().sum()) for i in range(0, n, step)))
    assert abs(float(norm) - total) <= 5 * 2.0 ** -24 * total
    c = 1.0 / (total + 1e-6)
    for i in range(0, n, step):
        want = g[i:i + step].double() * c
        assert bool(((out[i:i + step].double() - want).abs() <= (2.0 ** -8 + 6 * 2.0 ** -24) * want.abs() + 2.0 ** -134).all())


def test_resized_storage():
    """What a gradient's storage was resized to is not the clipper's memory any more."""
    g = rand(1000, torch.float32)
    clipper, into = L.GradClipper([g]), L.GradClipper([rand(1000, torch.float32)], [g])
    g.untyped_storage().resize_(0)
    for c in (clipper, into):
        with pytest.raises(RuntimeError, match="resized"):
            c.clip(1.0)
    g.untyped_storage().resize_(4000)
    g.fill_(1.0)
    assert abs(float(L.GradClipper([g]).clip(1.0)) - 1000 ** 0.5) < 1e-4
