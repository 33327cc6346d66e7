"""GPU tests of AdapterBank and AdapterBatch against the definition in 64 bits.

Tolerances.  y is rounded once (half a step of its type), u = scaling * A x is a
sum of K exact products in fp32, y a sum of R products more.  A sum of n terms
is off by n steps of 2^-23 of the sum of their magnitudes at most (tensor cores
cut instead of rounding), and a value of u that meets a 16-bit factor as two
16-bit parts is off by 2^-16 of itself (bf16; half a step of half a step).  So
with |Y| = |base| + sum_r |B_r| s sum_k |A_rk x_k|:

    |y - exact| <= eps / 2 |exact| + ((K + R + 16) 2^-23 + 2^-16) |Y|

and the gradients likewise, with the terms that their sums have."""

import pytest
import torch

import llm_quant_b200 as L

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def owners(ids, n, seq, num, counts=None):
    own = ids.long().cpu().repeat_interleave(seq)
    own[(own < 0) | (own >= num)] = -1
    if counts is not None:
        pos = torch.arange(n * seq) % max(seq, 1)
        own[pos >= counts.cpu().repeat_interleave(seq)] = -1
    return own


def reference(x, base, a, b, s, own, dy=None):
    """y and, with dy, dx, da, db in 64 bits, each with the sum of its terms' magnitudes."""
    x, a, b, s = x.double(), a.double(), b.double(), s.double()
    y = torch.zeros(x.shape[0], b.shape[2], dtype=torch.float64, device=x.device) if base is None else base.double().clone()
    ya = y.abs()
    out = [(y, ya)]
    if dy is not None:
        dy = dy.double()
        out += [(torch.zeros_like(t), torch.zeros_like(t)) for t in (x, a, b)]
    for i in range(a.shape[0]):
        rows = (own == i).nonzero().flatten().to(x.device)
        if not len(rows):
            continue
        xi = x[rows]
        u, ua = s[i] * xi @ a[i].T, s[i].abs() * xi.abs() @ a[i].abs().T
        y[rows] += u @ b[i]
        ya[rows] += ua @ b[i].abs()
        if dy is not None:
            d = dy[rows]
            v, va = s[i] * d @ b[i].T, s[i].abs() * d.abs() @ b[i].abs().T
            for (t, m), p, q in ((out[1], v @ a[i], va @ a[i].abs()),):
                t[rows], m[rows] = p, q
            out[2][0][i], out[2][1][i] = v.T @ xi, va.T @ xi.abs()
            out[3][0][i], out[3][1][i] = u.T @ d, ua.T @ d.abs()
    return out


def close(got, want, terms):
    want, mag = want
    eps = torch.finfo(got.dtype).eps
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -133
    tol = eps / 2 * want.abs() + ((terms + 16) * 2.0 ** -23 + 2.0 ** -16) * mag + tiny
    err = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((err <= tol).all()), f"worst {float((err / tol.clamp(min=1e-300)).max())} of the tolerance"


def make(n, seq, num, R, K, N, dt, seed=0, base=True, scale=1.0):
    g = torch.Generator(DEV).manual_seed(seed)

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)

    bank = L.AdapterBank(K, N, num, R, dtype=dt, device=DEV).requires_grad_(False)
    bank.lora_A.copy_(rand(num, R, K, scale=K ** -0.5))
    bank.lora_B.copy_(rand(num, R, N, scale=0.1))
    bank.scaling.copy_(torch.rand(num, generator=g, device=DEV) * 2 - 0.5)
    x = rand(n * seq, K, scale=scale)
    return bank, x, rand(n * seq, N) if base else None, rand(n * seq, N, scale=0.1)


# requests, tokens of each, adapters, rank, in, out
SHAPES = [
    (1, 1, 1, 1, 8, 8), (1, 1, 8, 16, 4096, 4096), (2, 1, 3, 16, 64, 128), (7, 1, 4, 4, 200, 72), (16, 1, 16, 64, 1032, 520),
    (33, 1, 5, 8, 264, 1288), (64, 1, 2, 24, 512, 256), (100, 1, 64, 33, 136, 2056), (200, 1, 7, 128, 256, 264),
    (1, 127, 2, 16, 128, 128), (1, 128, 1, 16, 256, 384), (1, 129, 3, 8, 72, 520), (3, 100, 2, 32, 1032, 248),
    (4, 333, 3, 64, 512, 1024), (2, 700, 1, 17, 264, 136), (5, 1, 8192, 2, 64, 64), (300, 3, 40, 16, 128, 1032),
    (1, 2500, 2, 128, 192, 320), (6, 513, 4, 12, 2056, 1160), (20, 260, 2, 16, 320, 256),
]


def some_ids(n, num, seed, none):
    g = torch.Generator().manual_seed(seed)
    lo = -1 if none else 0
    return torch.randint(lo, num, (n,), generator=g).to(torch.int32).to(DEV)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward(shape, dt):
    n, seq, num, R, K, N = shape
    bank, x, base, _ = make(n, seq, num, R, K, N, TYPES[dt])
    ids = some_ids(n, num, n + seq, n % 2)
    counts = torch.randint(0, seq + 1, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(5)).to(DEV) if seq > 2 else None
    batch = L.AdapterBatch(ids, num, seq, counts)
    own = owners(ids, n, seq, num, counts)
    for b in (base, None):
        y = bank(x, batch, b)
        close(y, reference(x, b, bank.lora_A, bank.lora_B, bank.scaling, own)[0], K + R)
        bare = (own < 0).to(DEV)
        assert torch.equal(y[bare], (b if b is not None else torch.zeros_like(y))[bare])
    kept = base.clone()
    assert torch.equal(bank.add_(kept, x, batch), bank(x, batch, base))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_backward(shape, dt):
    n, seq, num, R, K, N = shape
    bank, x, base, dy = make(n, seq, num, R, K, N, TYPES[dt], seed=1)
    bank.requires_grad_(True)
    ids = some_ids(n, num, n, n % 3 == 0)
    counts = torch.randint(0, seq + 1, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(6)).to(DEV) if seq > 2 else None
    batch = L.AdapterBatch(ids.long(), num, seq, counts)
    own = owners(ids, n, seq, num, counts)
    x.requires_grad_(True)
    base.requires_grad_(True)
    y = bank(x, batch, base)
    dx, da, db, dbase = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B, base), dy)
    with torch.no_grad():
        ry, rx, ra, rb = reference(x, base, bank.lora_A, bank.lora_B, bank.scaling, own, dy)
    most = max(int((own == i).sum()) for i in range(num))
    close(y.detach(), ry, K + R)
    close(dx, rx, N + R)
    close(da, ra, N + most)
    close(db, rb, K + most)
    assert torch.equal(dbase, dy)
    # equal calls, equal bits
    again = torch.autograd.grad(bank(x, batch, base), (x, bank.lora_A, bank.lora_B), dy)
    for p, q in zip((dx, da, db), again):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("R", [16, 32, 64, 128])
def test_many_tiles(R, dt):
    """Many tiles and columns to a block, of sequences that follow each other and
    of tokens in any order, with padding between them; calls that nothing waits between."""
    n, seq, num, K, N = 9, 515, 3, 136, 4360
    bank, x, base, dy = make(n, seq, num, R, K, N, TYPES[dt], seed=20)
    counts = torch.tensor([515, 512, 1, 0, 300, 515, 514, 129, 515], dtype=torch.int32, device=DEV)
    ids = torch.tensor([0, 1, 2, 0, -1, 1, 0, 2, 2], dtype=torch.int32, device=DEV)
    mixed = torch.randint(-1, num, (n * seq,), generator=torch.Generator().manual_seed(1)).int().to(DEV)
    batches = [(L.AdapterBatch(ids, num, seq, counts), owners(ids, n, seq, num, counts)),
               (L.AdapterBatch(mixed, num), owners(mixed, n * seq, 1, num))]
    for batch, own in batches:
        want = reference(x, base, bank.lora_A, bank.lora_B, bank.scaling, own)[0]
        got = [bank(x, batch, base) for _ in range(6)]
        close(got[0], want, K + R)
        kept = base.clone()
        assert torch.equal(bank.add_(kept, x, batch), got[0])
        assert all(torch.equal(got[0], y) for y in got)


def test_gradients_against_differences():
    """y is linear in x, in A and in B: a difference over any step is the
    derivative, up to the rounding of the two outputs."""
    dt = torch.float16
    bank, x, base, dy = make(5, 40, 3, 16, 256, 128, dt, seed=3)
    batch = L.AdapterBatch(some_ids(5, 3, 1, True), 3, 40)
    bank.requires_grad_(True)
    x.requires_grad_(True)
    grads = torch.autograd.grad(bank(x, batch), (x, bank.lora_A, bank.lora_B), dy)
    g = torch.Generator(DEV).manual_seed(9)
    for t, grad in zip((x, bank.lora_A, bank.lora_B), grads):
        step = torch.randn(t.shape, generator=g, device=DEV)
        with torch.no_grad():
            kept = t.detach().clone()
            sides = []
            moved = []
            for sign in (1, -1):
                t.copy_((kept.float() + sign * 0.5 * step * kept.float().std()).to(dt))
                moved.append(t.detach().double().clone())
                sides.append(bank(x, batch).double())
            t.copy_(kept)
        want = ((sides[0] - sides[1]) * dy.double()).sum()
        d = moved[0] - moved[1]
        got = (grad.double() * d).sum()
        half = torch.finfo(dt).eps / 2
        # each output and each gradient is off by half a step, and by the sums' share, which is below another half
        tol = 2 * half * (((sides[0].abs() + sides[1].abs()) * dy.double().abs()).sum() + (grad.double().abs() * d.abs()).sum())
        assert abs(float(want - got)) <= float(tol)


def test_fp32_parameters():
    """fp32 parameters are rounded to the activations' type; their gradients come in fp32."""
    dt = torch.bfloat16
    bank, x, base, dy = make(3, 50, 2, 8, 136, 264, dt, seed=4)
    bank = bank.float().requires_grad_(True)
    with torch.no_grad():
        bank.lora_A.add_(torch.randn_like(bank.lora_A) * 1e-4)
    ids = torch.tensor([0, 1, 0], device=DEV)
    batch = L.AdapterBatch(ids, 2, 50)
    y = bank(x, batch, base)
    da, db = torch.autograd.grad(y, (bank.lora_A, bank.lora_B), dy)
    assert da.dtype == db.dtype == torch.float32
    a, b = bank.lora_A.detach().to(dt), bank.lora_B.detach().to(dt)
    ry, _, ra, rb = reference(x, base, a, b, bank.scaling, owners(ids, 3, 50, 2), dy)
    close(y.detach(), ry, 136 + 8)
    close(da, ra, 264 + 100)
    close(db, rb, 136 + 100)


def test_subsets_of_gradients():
    bank, x, base, dy = make(4, 33, 2, 16, 128, 256, torch.bfloat16, seed=6)
    batch = L.AdapterBatch(some_ids(4, 2, 2, False), 2, 33)
    bank.requires_grad_(True)
    x.requires_grad_(True)
    whole = torch.autograd.grad(bank(x, batch, base), (x, bank.lora_A, bank.lora_B), dy)
    leaves = (x, bank.lora_A, bank.lora_B)
    for i, t in enumerate(leaves):
        for o in leaves:
            o.requires_grad_(o is t)
        got, = torch.autograd.grad(bank(x, batch, base), (t,), dy)
        assert torch.equal(got, whole[i])


def test_nothing_but_zeros_and_padding():
    """Adapters without tokens get zeros; a batch without adapters passes base on; padding may hold anything."""
    for dt in TYPES.values():
        bank, x, base, dy = make(3, 70, 4, 16, 128, 136, dt, seed=7)
        bank.requires_grad_(True)
        ids = torch.tensor([1, 3, 1], dtype=torch.int32, device=DEV)
        counts = torch.tensor([70, 0, 31], dtype=torch.int32, device=DEV)
        clean = bank(x, L.AdapterBatch(ids, 4, 70, counts), base)
        want = torch.autograd.grad(clean, (bank.lora_A, bank.lora_B), dy)
        bad, bad_dy = x.view(3, 70, -1).clone(), dy.view(3, 70, -1).clone()
        for t in (bad, bad_dy):
            t[1], t[2, 31:] = float("nan"), float("inf")
        bad = bad.view_as(x).requires_grad_(True)
        y = bank(bad, L.AdapterBatch(ids, 4, 70, counts), base)
        assert torch.equal(y, clean)
        dx, da, db = torch.autograd.grad(y, (bad, bank.lora_A, bank.lora_B), bad_dy.view_as(dy))
        assert torch.equal(da, want[0]) and torch.equal(db, want[1])
        for i in (0, 2, 3):
            assert not da[i].any() and not db[i].any()
        assert not dx.view(3, 70, -1)[1].any() and not dx.view(3, 70, -1)[2, 31:].any()
        none = L.AdapterBatch(torch.full((3,), -1, dtype=torch.int32, device=DEV), 4, 70)
        assert torch.equal(bank(x, none, base), base) and not bank(x, none).any()
        g = torch.autograd.grad(bank(x, none, base), (bank.lora_A, bank.lora_B), dy)
        assert not g[0].any() and not g[1].any()


def test_infinities_stay_in_their_rows():
    for dt in TYPES.values():
        bank, x, base, _ = make(1, 300, 1, 16, 128, 136, dt, seed=8)
        batch = L.AdapterBatch(torch.zeros(1, dtype=torch.int32, device=DEV), 1, 300)
        clean = bank(x, batch, base)
        bad = x.clone()
        bad[7, 3], bad[200, 64], bad[201, 127] = float("inf"), float("nan"), float("-inf")
        y = bank(bad, batch, base)
        rows = torch.ones(300, dtype=torch.bool, device=DEV)
        rows[[7, 200, 201]] = False
        assert torch.equal(y[rows], clean[rows])
        assert y[200].isnan().all() and not y[[7, 201]].isfinite().any()


@pytest.mark.parametrize("rows", [1, 40, 900])
def test_values_over_the_range_of_the_type(rows):
    """u may leave fp16's range in either direction; y does not."""
    dt = torch.float16
    K, N, R = 256, 136, 16
    bank, x, _, dy = make(rows, 1, 2, R, K, N, dt, seed=10)
    ids = some_ids(rows, 2, 3, False)
    batch = L.AdapterBatch(ids, 2)
    own = owners(ids, rows, 1, 2)
    for grow in (2.0 ** 12, 2.0 ** -14):
        with torch.no_grad():
            x2 = (x.float() * 200).to(dt) if grow > 1 else (x.float() * 2.0 ** -8).to(dt)
            bank.lora_A.copy_((torch.randn(2, R, K, device=DEV, generator=torch.Generator(DEV).manual_seed(1)) * min(grow, 600.0)).to(dt))
            bank.lora_B.copy_((torch.randn(2, R, N, device=DEV, generator=torch.Generator(DEV).manual_seed(2)) * (2.0 ** -13 if grow > 1 else 16.0)).to(dt))
            bank.scaling.fill_(1.0)
        bank.requires_grad_(True)
        y = bank(x2, batch)
        (ry, _, _, rb) = reference(x2, None, bank.lora_A.detach(), bank.lora_B.detach(), bank.scaling, own, dy)
        close(y.detach(), ry, K + R)
        small = (dy.float() * 2.0 ** -8).to(dt) if grow > 1 else dy
        db, = torch.autograd.grad(y, (bank.lora_B,), small)
        rb = reference(x2, None, bank.lora_A.detach(), bank.lora_B.detach(), bank.scaling, own, small)[3]
        if float(rb[0].abs().max()) < 60000:
            close(db, rb, K + rows)


def test_rows_of_other_strides():
    dt = torch.bfloat16
    bank, x, base, dy = make(3, 30, 2, 16, 128, 256, dt, seed=11)
    ids = some_ids(3, 2, 4, True)
    batch = L.AdapterBatch(ids, 2, 30)
    want = bank(x, batch, base)
    wide = torch.zeros(90, 400, dtype=dt, device=DEV)
    wide[:, 8:136] = x
    assert torch.equal(bank(wide[:, 8:136], batch, base), want)          # rows on 16 bytes: read as they are
    wide[:, 3:131] = x
    assert torch.equal(bank(wide[:, 3:131], batch, base), want)          # off them: copied
    assert torch.equal(bank(x.view(3, 30, 128), batch, base.view(3, 30, 256)).view(90, 256), want)
    assert torch.equal(bank(x.t().contiguous().t(), batch, base), want)
    y = torch.zeros(90, 264, dtype=dt, device=DEV)
    y[:, :256] = base
    bank.add_(y[:, :256], x, batch)
    assert torch.equal(y[:, :256], want) and not y[:, 256:].any()
    one = x[:1].expand(90, 128)                                          # rows that are all the same memory
    assert torch.equal(bank(one, batch, base), bank(one.contiguous(), batch, base))
    bank.requires_grad_(True)
    out = bank(x.clone().requires_grad_(True), batch, base)
    a = torch.autograd.grad(out.sum(), (bank.lora_A,), retain_graph=True)[0]  # dy is one value, expanded
    assert torch.equal(a, torch.autograd.grad(out, (bank.lora_A,), torch.ones_like(out))[0])
    out = bank(x, batch, base)
    turned = torch.autograd.grad(out, (bank.lora_A,), dy.t().contiguous().t(), retain_graph=True)[0]
    assert torch.equal(turned, torch.autograd.grad(out, (bank.lora_A,), dy)[0])


def test_no_tokens():
    bank = L.AdapterBank(64, 128, 3, 8, dtype=torch.bfloat16, device=DEV)
    batch = L.AdapterBatch(torch.zeros(0, dtype=torch.int32, device=DEV), 3)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = bank(x, batch)
    assert y.shape == (0, 128)
    dx, da, db = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), torch.zeros_like(y))
    assert dx.shape == (0, 64) and not da.any() and not db.any()
    batch = L.AdapterBatch(torch.zeros(4, dtype=torch.int32, device=DEV), 3, 0)
    assert bank(torch.zeros(4, 0, 64, dtype=torch.bfloat16, device=DEV), batch).shape == (4, 0, 128)


def test_captured_steps_and_new_requests():
    """A captured plan, forward and backward pass, replayed for other requests and values."""
    dt = torch.bfloat16
    for n, seq in ((6, 1), (5, 90)):
        bank, x, base, dy = make(n, seq, 3, 16, 256, 136, dt, seed=12)
        bank.requires_grad_(True)
        ids = some_ids(n, 3, 1, True)
        batch = L.AdapterBatch(ids, 3, seq)
        x.requires_grad_(True)

        def step():
            batch.update(ids)
            y = bank(x, batch, base)
            return [y.detach(), *torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), dy)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for seed in (2, 3):
            with torch.no_grad():
                ids.copy_(some_ids(n, 3, seed, True))
                x.copy_(torch.randn(x.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)))
            graph.replay()
            got = [t.clone() for t in held]
            for p, q in zip(got, step()):
                assert torch.equal(p, q)


def test_two_streams():
    """Calls of one bank on two streams at once, each with its own batch."""
    bank, x, base, _ = make(40, 20, 4, 16, 512, 520, torch.bfloat16, seed=13)
    batches = [L.AdapterBatch(some_ids(40, 4, s, True), 4, 20) for s in range(2)]
    want = [bank(x, b, base) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(bank(x, batches[i], base))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, y) for y in g)


def test_changed_plan_is_noticed():
    bank, x, base, dy = make(3, 5, 2, 8, 64, 64, torch.bfloat16)
    bank.requires_grad_(True)
    ids = some_ids(3, 2, 0, False)
    batch = L.AdapterBatch(ids, 2, 5)
    y = bank(x, batch, base)
    batch.update(ids)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward(dy)


def test_layers_and_their_step():
    """QLoRALinear with a bank: serving, a training step and the clipping of its
    gradients; a bank made of layers gives what the layers give."""
    torch.manual_seed(0)
    dt = torch.bfloat16
    K, N = 256, 384
    w = (torch.randn(N, K, device=DEV) * 0.05).to(dt)
    layers = []
    for r in (4, 16):
        ql = L.QLoRALinear(K, N, rank=r, alpha=2.0 * r).to(DEV)
        ql.pack_base(w)
        torch.nn.init.normal_(ql.lora_B, std=0.1)
        torch.nn.init.normal_(ql.bias, std=0.1)
        layers.append(ql)
    layers[1].bias = layers[0].bias
    bank = L.AdapterBank.from_layers(layers)
    x = torch.randn(2, 17, K, device=DEV).to(dt)
    batch = L.AdapterBatch(torch.tensor([1, 0], device=DEV), 2, 17)
    with torch.no_grad():
        y = layers[0](x, bank, batch)
        wf = layers[0]._dequantize_base().double()
        for i, owner in enumerate((1, 0)):
            ql = layers[owner]
            u = x[i].double() @ ql.lora_A.to(dt).double().T * ql.scaling
            low = u @ ql.lora_B.to(dt).double().T
            shared = x[i].double() @ wf.T + ql.bias.double()
            # the base product is rounded before the adapter is added: two roundings
            tol = 2.0 ** -8 * (shared.abs() + (shared + low).abs()) \
                + (K + 32) * 2.0 ** -23 * (x[i].double().abs() @ wf.abs().T + ql.bias.abs().double()) \
                + ((K + 32) * 2.0 ** -23 + 2.0 ** -16) * (2 * x[i].double().abs() @ ql.lora_A.to(dt).double().abs().T
                                                         @ ql.lora_B.to(dt).double().abs().T)
            assert bool(((y[i].double() - shared - low).abs() <= tol).all())
    ql = layers[0]
    ql.requires_grad_(False)
    before = ql(x)
    opt = torch.optim.SGD(bank.parameters(), lr=1e-2)
    out = ql(x, bank, batch)
    out.float().square().mean().backward()
    pipeline = L.QLoRA()
    grads = [p.grad.double().clone() for p in pipeline.trainable_params(bank)]
    norm = pipeline.clip_gradients(bank, 1e-3)
    want = torch.stack([g.square().sum() for g in grads]).sum().sqrt()
    assert abs(float(norm) - float(want)) <= 2.0 ** -23 * float(want)
    for p, g in zip(bank.parameters(), grads):
        assert bool(((p.grad.double() - g * (1e-3 / (want + 1e-6))).abs() <= 2.0 ** -8 * 1.001 * g.abs() * (1e-3 / want) + 1e-40).all())
    opt.step()
    assert torch.equal(ql(x), before)  # the layer's own adapter and base are as they were


def test_refusals_on_the_device():
    bank = L.AdapterBank(64, 128, 3, 8, dtype=torch.bfloat16, device=DEV)
    ids = torch.zeros(4, dtype=torch.int32, device=DEV)
    batch = L.AdapterBatch(ids, 3)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(TypeError, match="float32"):
        bank(x.float(), batch)
    with pytest.raises(RuntimeError, match="tokens"):
        bank(x[:3], batch)
    with pytest.raises(RuntimeError, match="features"):
        bank(torch.zeros(4, 72, dtype=torch.bfloat16, device=DEV), batch)
    with pytest.raises(RuntimeError, match="base"):
        bank(x, batch, torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV))
    with pytest.raises(ValueError, match="adapters"):
        bank(x, L.AdapterBatch(ids, 2))
    with pytest.raises(RuntimeError, match="no gradient"):
        bank.add_(torch.zeros(4, 128, dtype=torch.bfloat16, device=DEV), x, batch)
    with torch.no_grad(), pytest.raises(ValueError, match="16 bytes"):
        bank.add_(torch.zeros(4, 130, dtype=torch.bfloat16, device=DEV)[:, 1:129], x, batch)
    with torch.no_grad(), pytest.raises(ValueError, match="16 bytes"):
        bank.add_(torch.zeros(1, 128, dtype=torch.bfloat16, device=DEV).expand(4, 128), x, batch)
    with pytest.raises(TypeError, match="int32 or int64"):
        L.AdapterBatch(ids.float(), 3)
    with pytest.raises(ValueError, match="counts"):
        L.AdapterBatch(ids, 3, 2, ids.long())
    with pytest.raises(ValueError, match="counts"):
        L.AdapterBatch(ids, 3, 2, ids[:3])
    with pytest.raises(ValueError, match="num_adapters"):
        L.AdapterBatch(ids, 0)
    with pytest.raises(ValueError, match="expected 4"):
        batch.update(ids[:2])
    with pytest.raises(RuntimeError, match="CUDA"):
        L.AdapterBatch(ids.cpu(), 3)
    ql = L.QLoRALinear(64, 64).to(DEV)
    with pytest.raises(ValueError, match="together"):
        ql(x, bank)
    with pytest.raises(ValueError, match="beside"):
        ql(x, bank, batch)


def test_inference_mode():
    bank, x, base, _ = make(4, 1, 2, 8, 64, 64, torch.bfloat16)
    with torch.inference_mode():
        batch = L.AdapterBatch(torch.zeros(4, dtype=torch.int32, device=DEV), 2)
        y = base.clone()
        batch.update(torch.zeros(4, dtype=torch.int32, device=DEV))
        assert torch.equal(bank.add_(y, x, batch), bank(x, batch, base))


def test_gradient_of_b_alone_behind_another_bank():
    """The gradient of lora_B alone needs no product with dy first: its sums are the
    first launch of the backward pass, right behind the kernel that makes dy."""
    dt = torch.bfloat16
    first, x, _, _ = make(4, 1000, 2, 64, 128, 2048, dt, seed=30)
    second, _, _, dy = make(4, 1000, 2, 64, 2048, 1024, dt, seed=31)
    batch = L.AdapterBatch(some_ids(4, 2, 5, False), 2, 1000)
    first.lora_B.requires_grad_(True)
    between = first(x, batch)
    torch.cuda.synchronize()
    leaf = between.detach().requires_grad_(True)
    d, = torch.autograd.grad(second(leaf, batch), (leaf,), dy)
    torch.cuda.synchronize()
    want, = torch.autograd.grad(first(x, batch), (first.lora_B,), d)
    torch.cuda.synchronize()
    for _ in range(10):
        got, = torch.autograd.grad(second(first(x, batch), batch), (first.lora_B,), dy)
        assert torch.equal(got, want)


def test_types_of_a_module():
    """A bank whose module was moved to another type keeps its scaling in fp32;
    parameters in another 16-bit type than the activations are refused."""
    bank, x, base, _ = make(3, 1, 2, 8, 64, 64, torch.bfloat16, seed=32)
    bank.scaling.fill_(1.0 / 3.0)
    batch = L.AdapterBatch(torch.zeros(3, dtype=torch.int32, device=DEV), 2)
    want = bank(x, batch, base)
    bank.bfloat16()
    assert bank.scaling.dtype == torch.float32 and torch.equal(bank(x, batch, base), want)
    bank.half()
    with pytest.raises(TypeError, match="float16 for activations in bfloat16"):
        bank(x, batch, base)
    assert bank(x.half(), batch).dtype == torch.float16
    import copy
    assert torch.equal(copy.deepcopy(bank)(x.half(), batch), bank(x.half(), batch))


def test_infinities_stay_in_their_rows_of_tiles():
    """As above, where tokens share tiles (a call that keeps what its backward pass needs)."""
    for dt in TYPES.values():
        bank, x, base, _ = make(1, 300, 1, 16, 128, 136, dt, seed=8)
        bank.requires_grad_(True)
        batch = L.AdapterBatch(torch.zeros(1, dtype=torch.int32, device=DEV), 1, 300)
        clean = bank(x, batch, base).detach()
        bad = x.clone()
        bad[7, 3], bad[200, 64], bad[201, 127] = float("inf"), float("nan"), float("-inf")
        y = bank(bad, batch, base).detach()
        rows = torch.ones(300, dtype=torch.bool, device=DEV)
        rows[[7, 200, 201]] = False
        assert torch.equal(y[rows], clean[rows])
        assert y[200].isnan().all() and not y[[7, 201]].isfinite().any()


def test_in_place_on_its_own_input():
    """y may be x itself where the features agree."""
    for n, seq in ((5, 1), (3, 700)):
        bank, x, _, _ = make(n, seq, 2, 16, 256, 256, torch.bfloat16, seed=33)
        batch = L.AdapterBatch(some_ids(n, 2, 6, True), 2, seq)
        want = bank(x, batch, x)
        y = x.clone()
        assert torch.equal(bank.add_(y, y, batch), want)


def test_second_derivatives_are_refused():
    bank, x, base, dy = make(3, 5, 2, 8, 64, 64, torch.bfloat16)
    x.requires_grad_(True)
    y = bank(x, L.AdapterBatch(some_ids(3, 2, 0, False), 2, 5), base)
    with pytest.raises(RuntimeError, match="gradients of gradients"):
        torch.autograd.grad(y, (x,), dy, create_graph=True)


def test_captured_decode_step():
    """A captured call of few tokens, replayed for other requests."""
    bank, x, base, _ = make(8, 1, 4, 16, 512, 264, torch.bfloat16, seed=34)
    ids = some_ids(8, 4, 1, True)
    batch = L.AdapterBatch(ids, 4)
    bank(x, batch, base)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.update(ids)
        held = bank(x, batch, base)
    for seed in (2, 3):
        ids.copy_(some_ids(8, 4, seed, True))
        x.copy_(torch.randn(x.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(seed)))
        graph.replay()
        assert torch.equal(held, bank(x, L.AdapterBatch(ids, 4), base))


def test_nothing_ran_out():
    bank, x, base, _ = make(4, 300, 2, 16, 256, 256, torch.bfloat16)
    bank.requires_grad_(True)
    batch = L.AdapterBatch(some_ids(4, 2, 0, True), 2, 300)
    bank(x, batch, base).sum().backward()
    batch.check()


@pytest.mark.parametrize("seq", [1, 7, 32, 33, 200])
def test_plans(seq):
    """The plan's groups: every token once, in order, with its adapter."""
    for n, num in ((1, 1), (3, 2), (700, 5), (50, 200)):
        g = torch.Generator().manual_seed(n + seq)
        ids = torch.randint(-2, num + 2, (n,), generator=g)
        counts = torch.randint(-1, seq + 3, (n,), generator=g).int()
        for c in (None, counts):
            own = owners(ids, n, seq, num, None if c is None else c.clamp(0, seq))
            batch = L.AdapterBatch(ids.to(DEV), num, seq, None if c is None else c.to(DEV))
            t = n * seq
            plan = batch._plan.view(torch.int32).cpu()
            up = lambda k: (k + 3) // 4 * 4
            got_owner, order = plan[4:4 + t], plan[4 + up(t):4 + up(t) + t]
            assert torch.equal(got_owner.long(), own)
            key = torch.where(own < 0, num, own)
            assert torch.equal(order.long(), torch.sort(key, stable=True).indices)


def test_rows_of_other_strides_in_tiles():
    """Rows that are parts of wider ones, off 16 bytes, all the same memory, and
    turned, where tokens share tiles; sequences and tokens in any order."""
    dt = torch.float16
    n, seq, K, N = 3, 400, 128, 256
    bank, x, base, dy = make(n, seq, 2, 16, K, N, dt, seed=40)
    bank.requires_grad_(True)
    order = torch.randint(-1, 2, (n * seq,), generator=torch.Generator().manual_seed(3)).int().to(DEV)
    for batch in (L.AdapterBatch(some_ids(n, 2, 4, True), 2, seq), L.AdapterBatch(order, 2)):

        def step(x, base, dy):
            x = x.detach().requires_grad_(True)
            y = bank(x, batch, base)
            return [y.detach(), *torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), dy)]

        want = step(x, base, dy)
        wide, wide_b, wide_d = (torch.zeros(n * seq, w + 72, dtype=dt, device=DEV) for w in (K, N, N))
        for at in (8, 3):
            wide[:, at:at + K], wide_b[:, at:at + N], wide_d[:, at:at + N] = x, base, dy
            got = step(wide[:, at:at + K], wide_b[:, at:at + N], wide_d[:, at:at + N])
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        got = step(x.t().contiguous().t(), base.t().contiguous().t(), dy.t().contiguous().t())
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        same = [t[:1].expand_as(t) for t in (x, base, dy)]
        got, want = step(*same), step(*(t.contiguous() for t in same))
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_offsets_over_32_bits():
    """More than 2^31 values in base, out and dy."""
    dt = torch.bfloat16
    T, K, N, R = 151_000, 64, 14336, 8
    bank, x, _, _ = make(1, T, 2, R, K, N, dt, seed=41, base=False)
    bank.requires_grad_(True)
    batch = L.AdapterBatch(torch.tensor([1], device=DEV), 2, T)
    base = torch.empty(T, N, dtype=dt, device=DEV)
    for i in range(0, T, 10_000):
        base[i:i + 10_000].normal_(generator=torch.Generator(DEV).manual_seed(i))
    x.requires_grad_(True)
    y = bank(x, batch, base)
    dx, db = torch.autograd.grad(y, (x, bank.lora_B), base)
    y = y.detach()
    a, b, s = bank.lora_A[1].detach().double(), bank.lora_B[1].detach().double(), float(bank.scaling[1])
    sums, mags = torch.zeros(R, N, dtype=torch.float64, device=DEV), torch.zeros(R, N, dtype=torch.float64, device=DEV)
    for i in range(0, T, 10_000):
        xi, d = x.detach()[i:i + 10_000].double(), base[i:i + 10_000].double()
        u, ua = s * xi @ a.T, abs(s) * xi.abs() @ a.abs().T
        sums += u.T @ d
        mags += ua.T @ d.abs()
        close(y[i:i + 10_000], (d + u @ b, d.abs() + ua @ b.abs()), K + R)
        close(dx[i:i + 10_000], (s * d @ b.T @ a, abs(s) * d.abs() @ b.abs().T @ a.abs()), N + R)
    close(db[1], (sums, mags), K + T)
    assert not db[0].any()
    with torch.no_grad():
        assert torch.equal(bank.add_(base, x, batch), y)


def _off16(t):
    """A copy of t, side by side, whose address is off 16 bytes."""
    memory = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    memory[1:].copy_(t.detach().reshape(-1))
    return memory[1:].view(t.shape)


def _turned(t):
    return t.detach().transpose(0, -1).contiguous().transpose(0, -1)


@pytest.mark.parametrize("dt", TYPES)
def test_saved_tensors_that_come_back_laid_out_anew(dt):
    """Saved-tensor hooks may bring back copies: offloaded ones, dense ones of a
    strided x, turned ones, ones off 16 bytes.  Gradients are the same."""
    K, N = 128, 264
    bank, x, base, dy = make(2, 150, 2, 16, K, N, TYPES[dt], seed=50)
    bank.requires_grad_(True)
    batch = L.AdapterBatch(some_ids(2, 2, 3, False), 2, 150)
    wide = torch.zeros(300, 400, dtype=TYPES[dt], device=DEV)
    wide[:, 8:8 + K] = x
    rows = wide[:, 8:8 + K].requires_grad_(True)

    def grads(y):
        return torch.autograd.grad(y, (rows, bank.lora_A, bank.lora_B), dy)

    want = grads(bank(rows, batch, base))
    with torch.autograd.graph.save_on_cpu():
        y = bank(rows, batch, base)
    assert all(torch.equal(p, q) for p, q in zip(grads(y), want))
    packed = []

    def pack(t):
        packed.append(t.data_ptr())
        return t.detach()

    for unpack in (lambda t: t.contiguous().clone(), _turned, _off16):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = bank(rows, batch, base)
        assert all(torch.equal(p, q) for p, q in zip(grads(y), want))
    assert batch._plan.data_ptr() not in packed  # check() reads the plan that the kernels wrote to
    batch.check()
    for unpack, word in ((lambda t: t.cpu(), "came back on cpu"), (lambda t: t.double(), "came back in"),
                         (lambda t: t[:1], "other shapes")):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            y = bank(rows, batch, base)
        with pytest.raises(RuntimeError, match=word):
            grads(y)
    with torch.autograd.graph.save_on_cpu():
        y = bank(rows, batch, base)
    batch.update(some_ids(2, 2, 3, False))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        grads(y)


def test_a_batch_of_inference_mode_has_no_gradients():
    bank, x, base, _ = make(4, 1, 2, 8, 64, 64, torch.bfloat16)
    with torch.inference_mode():
        batch = L.AdapterBatch(torch.zeros(4, dtype=torch.int32, device=DEV), 2)
    assert torch.equal(bank(x, batch, base), bank(x, L.AdapterBatch(torch.zeros(4, dtype=torch.int32, device=DEV), 2), base))
    bank.requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference mode"):
        bank(x, batch, base)


def test_in_place_in_the_buffer_of_x():
    """Rows of y and of x in one buffer: columns beside each other, the same columns,
    tokens behind each other; rows of y that overlap other tokens' rows of x are refused."""
    for n, seq in ((5, 1), (3, 400)):
        T, K, N = n * seq, 128, 64
        bank, x, base, _ = make(n, seq, 2, 16, K, N, torch.bfloat16, seed=51)
        batch = L.AdapterBatch(some_ids(n, 2, 6, True), 2, seq)
        want = bank(x, batch, base)

        def placed(cols, xs, ys):
            buf = torch.zeros(2 * T + 2, cols, dtype=torch.bfloat16, device=DEV)
            vx, vy = buf[xs[0]:xs[0] + T, xs[1]:xs[1] + K], buf[ys[0]:ys[0] + T, ys[1]:ys[1] + N]
            vx.copy_(x)
            vy.copy_(base)
            return vx, vy

        for at in (((0, 0), (0, 128)), ((0, 64), (0, 0)), ((0, 0), (1, 128)), ((1, 0), (0, 128)), ((0, 0), (T, 0)), ((T, 8), (0, 72))):
            vx, vy = placed(192, *at)
            assert torch.equal(bank.add_(vy, vx, batch), want)
        for c in (0, 8, 64):  # columns of x itself
            vx, vy = placed(K, (0, 0), (0, c))
            mine = bank(vx, batch, vy)
            assert torch.equal(bank.add_(vy, vx, batch), mine)
        for cols, xs, ys in ((K, (0, 0), (1, 0)), (K, (1, 0), (0, 64)), (192, (0, 0), (1, 64)), (192, (1, 0), (0, 64))):
            vx, vy = placed(cols, xs, ys)
            with pytest.raises(ValueError, match="overlap other tokens"):
                bank.add_(vy, vx, batch)
        flat = torch.zeros(T * K, dtype=torch.bfloat16, device=DEV)  # other distances from row to row
        with pytest.raises(ValueError, match="overlap other tokens"):
            bank.add_(flat[:T * N].view(T, N), flat.view(T, K), batch)
        with pytest.raises(ValueError, match="overlap other tokens"):  # windows of x that overlap each other
            bank.add_(flat.as_strided((T, N), (64, 1), 0), flat.as_strided((T, K), (64, 1), 0), batch)
        one, first = x[:1], L.AdapterBatch(torch.zeros(1, dtype=torch.int32, device=DEV), 2)
        mine = bank(one, first, one[:, 8:72])
        assert torch.equal(bank.add_(one[:, 8:72], one, first), mine)


class _Twice(torch.nn.Module):
    def forward(self, t):
        return 2 * t


def test_parametrized_banks_and_hooks():
    """Tensors that are computed from others, and what hooks and wrappers do around a bank's call."""
    dt = torch.bfloat16
    bank, x, base, dy = make(3, 20, 2, 16, 128, 256, dt, seed=52)
    batch = L.AdapterBatch(some_ids(3, 2, 4, True), 2, 20)
    plain, _, _, _ = make(3, 20, 2, 16, 128, 256, dt, seed=52)
    plain.lora_A.mul_(2)
    for b in (bank, plain):
        b.requires_grad_(True)
    torch.nn.utils.parametrize.register_parametrization(bank, "lora_A", _Twice())
    y, want = bank(x, batch, base), plain(x, batch, base)
    assert torch.equal(y, want)
    got = torch.autograd.grad(y, (bank.parametrizations.lora_A.original, bank.lora_B), dy)
    ref = torch.autograd.grad(want, (plain.lora_A, plain.lora_B), dy)
    assert torch.equal(got[0], 2 * ref[0]) and torch.equal(got[1], ref[1])

    class Wrapped(torch.nn.Module):
        in_features, out_features = 128, 256

        def __init__(self):
            super().__init__()
            self.bank, self.calls = plain, 0

        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                return getattr(super().__getattr__("bank"), name)

        def forward(self, *args):
            self.calls += 1
            return self.bank(*args)

    ql = L.QLoRALinear(128, 256).to(DEV)
    ql.pack_base((torch.randn(256, 128, device=DEV, generator=torch.Generator(DEV).manual_seed(0)) * 0.1).to(dt))
    wrapped, seen = Wrapped(), []
    with torch.no_grad():
        want = ql(x, plain, batch)
        assert torch.equal(ql(x, wrapped, batch), want) and wrapped.calls == 1
        hooks = [plain.register_forward_pre_hook(lambda m, args: seen.append("before")),
                 plain.register_forward_hook(lambda m, args, out: seen.append("behind"))]
        assert torch.equal(ql(x, plain, batch), want) and seen == ["before", "behind"]
        for h in hooks:
            h.remove()
        every = torch.nn.modules.module.register_module_forward_hook(lambda m, args, out: seen.append(type(m)))
        assert torch.equal(ql(x, plain, batch), want) and L.AdapterBank in seen
        every.remove()


def test_check_waits_for_other_streams():
    """The status of work that is still on its way on a stream of its own (here a copy in its place) is waited for."""
    batch = L.AdapterBatch(torch.zeros(4, dtype=torch.int32, device=DEV), 2)
    batch.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
        batch._plan[:4].view(torch.int32).fill_(7)
    with pytest.raises(RuntimeError, match="ran out"):
        batch.check()
    batch.update(torch.zeros(4, dtype=torch.int32, device=DEV))
    batch.check()


def whole_numbers(n, seq, num, R, K, N, dt, seed, most=2):
    """As make, in small whole numbers, whose products and sums fp32 holds exactly (scaling: powers of two)."""
    g = torch.Generator(DEV).manual_seed(seed)

    def rand(*shape):
        return torch.randint(-most, most + 1, shape, generator=g, device=DEV).to(dt)

    bank = L.AdapterBank(K, N, num, R, dtype=dt, device=DEV).requires_grad_(False)
    bank.lora_A.copy_(rand(num, R, K))
    bank.lora_B.copy_(rand(num, R, N))
    bank.scaling.copy_(2.0 ** torch.randint(-1, 2, (num,), generator=g, device=DEV).float())
    return bank, rand(n * seq, K), rand(n * seq, N), rand(n * seq, N)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("R", [5, 16, 64, 128])
def test_infinities_in_gradients(R, dt):
    """Infinite x and dy: gradients are infinite with the sign, and no numbers,
    where the definition's are, in every form of a run; the others are as without
    them.  (Whole numbers: sums are exact, signs and zeros certain.)"""
    t = TYPES[dt]
    n, seq, num, K, N = 6, 333, 3, 136, 264
    bank, x, base, dy = whole_numbers(n, seq, num, R, K, N, t, seed=60)
    bank.scaling.abs_()
    bank = bank.float().requires_grad_(True)  # gradients in fp32: exact
    inf = float("inf")
    ids = torch.tensor([0, 2, 0, -1, 0, 2], dtype=torch.int32, device=DEV)
    mixed = torch.randint(-1, num, (n * seq,), generator=torch.Generator().manual_seed(4)).int().to(DEV)
    for batch, own in ((L.AdapterBatch(ids, num, seq), owners(ids, n, seq, num)),
                       (L.AdapterBatch(mixed, num), owners(mixed, n * seq, 1, num))):
        bad, bad_dy = x.clone(), dy.clone()
        for row, column, value in ((7, 3, inf), (200, 64, -inf), (350, 100, inf), (1500, 100, -inf), (1700, 3, inf)):
            bad[row, column] = value
        for row, column, value in ((9, 17, -inf), (800, 33, inf), (801, 33, -inf), (1999 - 2, 263, inf)):
            bad_dy[row, column] = value
        for p, d in ((x, dy), (bad, dy), (x, bad_dy), (bad, bad_dy)):
            y = bank(p, batch, base)
            da, db = torch.autograd.grad(y, (bank.lora_A, bank.lora_B), d)
            with torch.no_grad():
                _, _, (ra, _), (rb, _) = reference(p, base, bank.lora_A, bank.lora_B, bank.scaling, own, d)
            for got, want in ((da, ra), (db, rb)):
                nan = want.isnan()
                assert torch.equal(got.isnan(), nan)
                assert torch.equal(got[~nan].double(), want[~nan])
        batch.check()


def test_small_values_beside_great_ones():
    """fp16: what meets a factor in two parts is off by 2^-22 of itself or, beside
    much greater values, by 2^-37 of the greatest: of a token's ranks in y and dx,
    of an adapter's tokens in the gradients.  Columns that are zero where the great
    values are show the small ones alone."""
    dt = torch.float16
    n, seq, R, K, N = 2, 400, 16, 136, 264
    bank, x, base, dy = make(n, seq, 2, R, K, N, dt, seed=61)
    T = n * seq
    own = owners(torch.tensor([1, 0]), n, seq, 2)
    batch = L.AdapterBatch(torch.tensor([1, 0], device=DEV), 2, seq)
    # tokens by 2^-18 to 2^8 of dy, ranks by 2^-20 to 1 of A and B (within fp16's normal numbers after their own sizes)
    size = 2.0 ** -torch.randint(-8, 10, (T, 1), device=DEV, generator=torch.Generator(DEV).manual_seed(1)).double()
    great = size.flatten() > 16
    dy = (dy.double() * size).to(dt)
    x = (x.double() * size.clamp(max=16)).to(dt)
    x[great, :40] = 0
    dy[great, :40] = 0
    ranks = 2.0 ** -torch.arange(0, R, device=DEV).double()[None, :, None] / 4
    with torch.no_grad():
        bank.lora_A.copy_(bank.lora_A.double() * ranks * 8)
        bank.lora_B.copy_(bank.lora_B.double() * ranks * 8)
        bank.lora_A[:, :4, 60:90] = 0  # the great ranks have no part in these columns
        bank.lora_B[:, :4, 60:90] = 0
    bank = bank.float().requires_grad_(True)
    x.requires_grad_(True)
    y = bank(x, batch)
    dx, da, db = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), dy)
    with torch.no_grad():
        a, b, s = bank.lora_A.double(), bank.lora_B.double(), bank.scaling.double()
        ry, rx, ra, rb = reference(x, None, a, b, bank.scaling, own, dy)
        o = own.to(DEV)
        u = torch.einsum("tk,trk->tr", x.double(), a[o]) * s[o][:, None]
        v = torch.einsum("tn,trn->tr", dy.double(), b[o]) * s[o][:, None]

        def check(got, want, terms, far):
            half, tiny = (2.0 ** -11, 2.0 ** -25) if got.dtype == dt else (2.0 ** -24, 2.0 ** -133)
            exact, mag = want
            tol = half * exact.abs() + ((terms + 16) * 2.0 ** -23 + 2.0 ** -22) * mag + 2.0 ** -37 * far + tiny
            err = (got.double() - exact).abs()
            assert bool((err <= tol).all()), f"worst {float((err / tol).max())} of the tolerance"

        check(y.detach(), ry, K + R, u.abs().amax(1, keepdim=True) * b.abs().sum(1)[o])
        check(dx, rx, N + R, v.abs().amax(1, keepdim=True) * a.abs().sum(1)[o])
        for got, want, terms, low, rows in ((da, ra, N, v, x), (db, rb, K, u, dy)):
            far = torch.stack([low[o == i].abs().max() * rows.detach().double()[o == i].abs().sum(0) for i in range(2)])[:, None]
            check(got, want, terms + seq, far)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_whole_numbers(shape, dt):
    """Small whole numbers: every product and every sum is exact in fp32 (and u and v
    in two parts), in whatever order, so that y and dx are the definition's,
    rounded once, and gradients in fp32 are the definition's."""
    n, seq, num, R, K, N = shape
    t = TYPES[dt]
    bank, x, base, dy = whole_numbers(n, seq, num, R, K, N, t, seed=62)
    bank = bank.float().requires_grad_(True)
    ids = some_ids(n, num, n, n % 3 == 0)
    counts = torch.randint(0, seq + 1, (n,), dtype=torch.int32, generator=torch.Generator().manual_seed(6)).to(DEV) if seq > 2 else None
    batch = L.AdapterBatch(ids, num, seq, counts)
    x.requires_grad_(True)
    y = bank(x, batch, base)
    dx, da, db = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), dy)
    with torch.no_grad():
        served = bank(x, batch, base)
        (ry, _), (rx, _), (ra, _), (rb, _) = reference(x, base, bank.lora_A, bank.lora_B, bank.scaling,
                                                       owners(ids, n, seq, num, counts), dy)
    for low, w in ((x.detach().float() @ bank.lora_A.detach().flatten(0, 1).T, "u"), (dy.float() @ bank.lora_B.detach().flatten(0, 1).T, "v")):
        assert float(low.abs().max()) * 2 < 2 ** 14, w  # halves of up to twice that: 16 bits
    assert max(float(g.abs().max()) for g in (ra, rb)) < 2 ** 22
    for got, want in ((y, ry), (served, ry), (dx, rx)):
        assert torch.equal(got.detach(), want.to(t))
    assert torch.equal(da.double(), ra) and torch.equal(db.double(), rb)


def test_whole_numbers_over_32_bits():
    """As above, with more than 2^31 values in base, out and dy."""
    dt = torch.bfloat16
    T, K, N, R = 151_000, 64, 14336, 8
    bank, x, base, _ = whole_numbers(1, T, 2, R, K, N, dt, seed=63)
    bank = bank.float().requires_grad_(True)
    batch = L.AdapterBatch(torch.tensor([1], device=DEV), 2, T)
    x.requires_grad_(True)
    y = bank(x, batch, base)
    dx, da, db = torch.autograd.grad(y, (x, bank.lora_A, bank.lora_B), base)
    y = y.detach()
    a, b, s = bank.lora_A[1].detach().double(), bank.lora_B[1].detach().double(), float(bank.scaling[1])
    ra, rb = torch.zeros(R, K, dtype=torch.float64, device=DEV), torch.zeros(R, N, dtype=torch.float64, device=DEV)
    for i in range(0, T, 10_000):
        xi, d = x.detach()[i:i + 10_000].double(), base[i:i + 10_000].double()
        u, v = s * xi @ a.T, s * d @ b.T
        ra += v.T @ xi
        rb += u.T @ d
        assert torch.equal(y[i:i + 10_000], (d + u @ b).to(dt))
        assert torch.equal(dx[i:i + 10_000], (v @ a).to(dt))
    assert torch.equal(da[1].double(), ra) and torch.equal(db[1].double(), rb)
    assert not da[0].any() and not db[0].any()


def test_checkpointed_calls():
    """Activation checkpointing: what the forward call saved is computed again in the backward pass."""
    from torch.utils.checkpoint import checkpoint
    bank, x, base, dy = make(3, 70, 2, 16, 128, 256, torch.bfloat16, seed=64)
    bank.requires_grad_(True)
    x.requires_grad_(True)
    batch = L.AdapterBatch(some_ids(3, 2, 4, True), 2, 70)
    leaves = (x, bank.lora_A, bank.lora_B)
    want = torch.autograd.grad(bank(x, batch, base), leaves, dy)
    got = torch.autograd.grad(checkpoint(bank, x, batch, base, use_reentrant=False), leaves, dy)
    checkpoint(bank, x, batch, base, use_reentrant=True).backward(dy)
    for p, q, w in zip(got, leaves, want):
        assert torch.equal(p, w) and torch.equal(q.grad, w)


def test_a_flag_of_infinities_changes_nothing_later():
    """A plan keeps that a call with it had sums that are no number; its later calls give what they give without."""
    bank, x, base, dy = make(4, 300, 2, 24, 136, 264, torch.float16, seed=65)
    bank.requires_grad_(True)
    ids = some_ids(4, 2, 4, True)
    leaves = (bank.lora_A, bank.lora_B)
    want = torch.autograd.grad(bank(x, L.AdapterBatch(ids, 2, 300), base), leaves, dy)
    batch = L.AdapterBatch(ids, 2, 300)
    bad = x.clone()
    bad[torch.arange(0, 1200, 7), 3] = float("inf")
    assert not torch.autograd.grad(bank(bad, batch, base), leaves, dy)[0].isfinite().all()
    for _ in range(2):
        got = torch.autograd.grad(bank(x, batch, base), leaves, dy)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
