"""ash.linear, ash.rms_norm, ash.QuantizedRows and ash.FeatureDecoder against their
formulas in 64 bits (layers_reference.py, where the tolerances are derived)."""
import pytest
import torch

import layers_reference as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ids = lambda t: str(t).replace("torch.", "")


def rand(g, *shape, size=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * size).to(dtype).to(DEV)


def operands(rows, k, m, dtype, seed=0, a=1.0, sine=False):
    g = torch.Generator().manual_seed(1000 + seed)
    size = k**-0.5 * (1.4 / a if sine else 1.0)
    x, w, b = rand(g, rows, k, dtype=dtype), rand(g, m, k, size=size, dtype=dtype), rand(g, m, size=size, dtype=dtype)
    return x, w, b, rand(g, rows, m, dtype=dtype), rand(g, rows, m, dtype=dtype), rand(g, rows, k, dtype=dtype)


def leaves(*tensors):
    return [t.detach().requires_grad_() for t in tensors]


# one row to several tiles, every tail of a chunk, a step and a tile
SHAPES = [(1, 1, 1), (1, 64, 64), (5, 3, 2), (16, 131, 33), (17, 8, 31), (64, 256, 100), (65, 19, 64), (127, 64, 1),
          (130, 67, 129), (300, 200, 257), (1000, 33, 65), (2049, 64, 64), (4100, 19, 128), (777, 40, 24),
          (513, 24, 50), (40000, 31, 30), (9000, 70, 90), (17000, 67, 33), (6000, 300, 130), (300, 40, 5000), (3, 17, 65536)]
ACTS = [("none", 1.0), ("relu", 1.0), ("silu", 1.0), ("gelu", 1.0), ("softplus", 100.0), ("sine", 30.0)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_linear_and_its_gradients(gpu_ash, shape, dtype):
    rows, k, m = shape
    kind, a = ACTS[sum(shape) % len(ACTS)]
    x, w, b, r, gy, _ = operands(rows, k, m, dtype, a=a, sine=kind == "sine")
    y, d, _, _ = ref.linear(x, w, b, kind, a, r)
    ref.check(gpu_ash.linear(x, w, b, activation=kind, scale=a, residual=r), y, dtype, "forward")
    gx, gw, gb, _ = ref.linear_gradients(gy, x, w, d, kind, dtype)
    lx, lw, lb, lr = leaves(x, w, b, r)
    out = gpu_ash.linear(lx, lw, lb, activation=kind, scale=a, residual=lr)
    ref.check(out, y, dtype, "forward that learns")
    got = torch.autograd.grad(out, [lx, lw, lb, lr], gy)
    for have, want, what in zip(got, (gx, gw, gb, ref.Off(gy)), ("gx", "gw", "gb", "gr")):
        ref.check(have, want, dtype, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("rows,k,m,kind", [(16640, 1032, 1000, "gelu"), (20001, 520, 776, "none"),
                                           (33000, 256, 512, "sine"), (4100, 2056, 544, "silu"),
                                           (10007, 136, 264, "softplus"), (2500, 1032, 1000, "relu"), (3333, 80, 104, "none")])
def test_linear_and_its_gradients_in_large_tiles(gpu_ash, rows, k, m, kind, dtype):
    """Sizes that end inside a tile and inside a step, an odd number of steps; aligned
    and not (the other tiles take those)."""
    a = 30.0 if kind == "sine" else 1.0
    x, w, b, r, gy, _ = operands(rows, k + 1, m, dtype, seed=20, a=a, sine=kind == "sine")
    w, wide = w[:, :k].contiguous(), torch.cat([x, x[:, :7]], 1)
    for x in (x[:, :k].contiguous(), wide[:, :k], x[:, 1:]):
        y, d, _, _ = ref.linear(x, w, b, kind, a, r)
        gx, gw, gb, _ = ref.linear_gradients(gy, x, w, d, kind, dtype)
        lx, lw, lb = leaves(x, w, b)
        out = gpu_ash.linear(lx, lw, lb, activation=kind, scale=a, residual=r)
        ref.check(out, y, dtype, "forward")
        got = torch.autograd.grad(out, [lx, lw, lb], gy)
        for have, want, what in zip(got, (gx, gw, gb), ("gx", "gw", "gb")):
            ref.check(have, want, dtype, what)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=ids)
@pytest.mark.parametrize("rows,k,m", [(16640, 136, 1000), (4100, 136, 264), (16500, 72, 1004)])
def test_residuals_of_large_tiles(gpu_ash, rows, k, m, dtype):
    """Of rows that lie apart, at addresses that are not aligned, that broadcast; of
    8-bit operands too."""
    x, w, b, wide, _, _ = operands(rows, k, m, dtype, seed=21)
    y, _, _, _ = ref.linear(x, w, b, "gelu", 1.0)
    apart = torch.cat([wide, wide[:, :16]], 1)
    q = [gpu_ash.QuantizedRows.of(t) for t in (x, w)]
    of8, _, _, _ = ref.linear(q[0].data.float(), q[1].data.float(), b, "silu", 1.0, None, q[0].scales, q[1].scales, True)
    for r in (wide, apart[:, 8:m + 8], apart[:, 3:m + 3], wide[:1].expand(rows, m), wide[5], wide[:, :1]):
        more = r.expand(rows, m).double()
        ref.check(gpu_ash.linear(x, w, b, activation="gelu", residual=r), y + ref.Off(more), dtype)
        ref.check(gpu_ash.linear(*q, b, activation="silu", residual=r), of8 + ref.Off(more), dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("kind,a", ACTS)
def test_activations(gpu_ash, kind, a, dtype):
    """Arguments over the whole range, far tails among them; no bias, no residual."""
    z = torch.cat([torch.linspace(-30, 30, 4001), torch.tensor([0.0, -0.0, 88.0, -88.0, 1e4, -1e4, 1e-30])])
    if kind == "sine":
        z = z / 3
    x = z.to(dtype).to(DEV).reshape(-1, 1)
    w = torch.ones(1, 1, dtype=dtype, device=DEV)
    y, d, _, _ = ref.linear(x, w, None, kind, a)
    lx, = leaves(x)
    out = gpu_ash.linear(lx, w, activation=kind, scale=a)
    ref.check(out, y, dtype, "f")
    gx, = torch.autograd.grad(out, lx, torch.ones_like(out))
    ref.check(gx, ref.linear_gradients(torch.ones_like(out), x, w, d, kind, dtype)[0], dtype, "f'")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("kind,a", ACTS)
@pytest.mark.parametrize("shape", [(3, 5, 4), (200, 67, 129), (1030, 64, 64), (700, 20, 50), (40000, 50, 20)], ids=str)
def test_second_order(gpu_ash, shape, kind, a, dtype):
    x, w, b, _, gy, u = operands(*shape, dtype, seed=1, a=a, sine=kind == "sine")
    _, d, dd, _ = ref.linear(x, w, b, kind, a)
    gx, _, _, gz = ref.linear_gradients(gy, x, w, d, kind, dtype)
    lx, lw, lb, lg = leaves(x, w, b, gy)
    got_x, = torch.autograd.grad(gpu_ash.linear(lx, lw, lb, activation=kind, scale=a), lx, lg, create_graph=True)
    ref.check(got_x, gx, dtype, "gx")
    want = ref.linear_second(gy, x, w, d, dd, gz, kind, dtype, u)
    for have, one, what in zip(torch.autograd.grad(got_x, [lg, lx, lw, lb], u), want, ("gy", "x", "w", "b")):
        ref.check(have, one, dtype, what)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("asked", ["wb", "xwb", "w", "b", "xw"])
def test_second_order_of_the_gradients_of_weight_and_bias(gpu_ash, asked, dtype):
    rows, k, m = 333, 40, 70
    x, w, b, _, gy, u = operands(rows, k, m, dtype, seed=2)
    g = torch.Generator().manual_seed(3)
    ups = {"x": u, "w": rand(g, m, k, dtype=dtype), "b": rand(g, m, dtype=dtype)}
    _, d, dd, _ = ref.linear(x, w, b, "silu")
    gz = ref.linear_gradients(gy, x, w, d, "silu", dtype)[3]
    lx, lw, lb, lg = leaves(x, w, b, gy)
    of = dict(x=lx, w=lw, b=lb)
    firsts = torch.autograd.grad(gpu_ash.linear(lx, lw, lb, activation="silu"), [of[n] for n in asked], lg, create_graph=True)
    got = torch.autograd.grad(firsts, [lg, lx, lw, lb], [ups[n] for n in asked])
    want = ref.linear_second(gy, x, w, d, dd, gz, "silu", dtype, *[ups[n] if n in asked else None for n in "xwb"])
    for have, one, what in zip(got, want, ("gy", "x", "w", "b")):
        ref.check(have, one, dtype, what)


def test_gradients_against_differences(gpu_ash):
    """Of a loss through two layers and a norm, first order and that of an eikonal
    term, along a direction: central differences of the plain form in 64 bits."""
    g = torch.Generator().manual_seed(5)
    names = ("x", "w1", "b1", "n", "w2", "b2")
    p = [rand(g, 50, 19), rand(g, 40, 19, size=0.3), rand(g, 40, size=0.1), rand(g, 40), rand(g, 3, 40, size=0.3), rand(g, 3)]
    p64 = [t.double() for t in p]
    way = [rand(g, *t.shape).double() for t in p]

    def plain(x, w1, b1, n, w2, b2):
        z = x @ w1.t() + b1
        h = torch.nn.functional.softplus(10 * z) / 10
        s = h + x[:, :1]
        h = s / (s.square().mean(1, keepdim=True) + 1e-6).sqrt() * n
        return torch.sin(2 * (h @ w2.t() + b2))

    def own(x, w1, b1, n, w2, b2):
        h = gpu_ash.linear(x, w1, b1, activation="softplus", scale=10.0)
        h, _ = gpu_ash.rms_norm(h, n, residual=x[:, :1])
        return gpu_ash.linear(h, w2, b2, activation="sine", scale=2.0)

    def loss(f, p):
        x = p[0]
        y = f(*p)
        gx, = torch.autograd.grad(y[:, 0].sum(), x, create_graph=True)
        return y.square().sum() + (gx.norm(dim=1) - 1).square().sum()

    l32 = leaves(*p)
    total = loss(own, l32)
    got = torch.autograd.grad(total, l32)
    h = 1e-5
    at = lambda s, n=None: float(loss(plain, leaves(*[t + s * v if n in (None, i) else t for i, (t, v) in enumerate(zip(p64, way))])))
    assert abs(float(total.detach()) - at(0)) <= 1e-5 * abs(at(0))
    for i, name in enumerate(names):
        slope = (at(h, i) - at(-h, i)) / (2 * h)
        have = float((got[i].double() * way[i]).sum())
        size = float((got[i].double() * way[i]).abs().sum())
        # float32 through a dozen operations of up to 50 terms: 2^-24 * 12 * 50 of the terms' magnitudes
        assert abs(have - slope) <= 4e-5 * size + 1e-6 * abs(slope), name


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_layouts(gpu_ash, dtype):
    """Rows that are parts of wider rows (no alignment), rows that lie across, a
    weight that lies across, residuals and gradients that broadcast, more axes."""
    g = torch.Generator().manual_seed(7)
    wide = rand(g, 70, 90, dtype=dtype)
    x, across = wide[:, 1:68], rand(g, 67, 70, dtype=dtype).t()
    w = rand(g, 67, 48, size=0.1, dtype=dtype).t()
    b = rand(g, 96, dtype=dtype)[::2]
    for rows in (x, across, x[:1].expand(70, 67), x[::3], x[3]):
        for residual in (None, rand(g, 48, dtype=dtype), rand(g, 70, 1, dtype=dtype)[: rows.shape[0] if rows.dim() == 2 else 1],
                         rand(g, 1, dtype=dtype)):
            if rows.dim() == 1 and residual is not None and residual.dim() == 2:
                continue
            flat = rows.reshape(-1, 67)
            more = None if residual is None else residual.expand(*rows.shape[:-1], 48).reshape(-1, 48)
            y, d, _, _ = ref.linear(flat, w, b, "gelu", 1.0, more)
            ref.check(gpu_ash.linear(rows, w, b, activation="gelu", residual=residual).reshape(-1, 48), y, dtype)
            lx, lw, lb = leaves(rows, w, b)
            lr = None if residual is None else residual.detach().requires_grad_()
            out = gpu_ash.linear(lx, lw, lb, activation="gelu", residual=lr)
            assert out.shape == (*rows.shape[:-1], 48)
            one = torch.ones((), dtype=dtype, device=DEV).expand_as(out)   # as sum() gives it
            got = torch.autograd.grad(out, [lx, lw, lb] + ([] if lr is None else [lr]), one)
            gx, gw, gb, _ = ref.linear_gradients(one.reshape(-1, 48), flat, w, d, "gelu", dtype)
            ref.check(got[0].reshape(-1, 67), gx, dtype)
            ref.check(got[1], gw, dtype)
            ref.check(got[2], gb, dtype)
            if lr is not None:
                assert got[3].shape == lr.shape and float(got[3].sum()) == flat.shape[0] * 48
    x4 = rand(g, 2, 3, 5, 67, dtype=dtype)
    y, _, _, _ = ref.linear(x4.reshape(-1, 67), w, None)
    out = gpu_ash.linear(x4, w)
    assert out.shape == (2, 3, 5, 48)
    ref.check(out.reshape(-1, 48), y, dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_no_rows(gpu_ash, dtype):
    x, w, b = leaves(torch.empty(0, 20, dtype=dtype, device=DEV), torch.ones(9, 20, dtype=dtype, device=DEV),
                     torch.ones(9, dtype=dtype, device=DEV))
    out = gpu_ash.linear(x, w, b, activation="silu")
    assert out.shape == (0, 9)
    gx, gw, gb = torch.autograd.grad(out.sum(), [x, w, b])
    assert gx.shape == (0, 20) and not gw.any() and not gb.any()
    n = torch.ones(20, dtype=dtype, device=DEV, requires_grad=True)
    out, total = gpu_ash.rms_norm(x, n, residual=x.detach())
    gx, gn = torch.autograd.grad(out.sum() + total.sum(), [x, n])
    assert out.shape == total.shape == gx.shape == (0, 20) and not gn.any()
    q = gpu_ash.rms_norm(x.detach(), quantize=True)
    assert q.data.shape == (0, 20) and q.scales.shape == (0,)
    assert gpu_ash.linear(q, gpu_ash.QuantizedRows.of(w)).shape == (0, 9)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_what_is_not_finite_stays_in_its_row(gpu_ash, dtype):
    for rows in (8, 200):
        x, w, b, r, _, _ = operands(rows, 70, 40, dtype, seed=8)
        plain = gpu_ash.linear(x, w, b, residual=r)
        x[3, 5], x[5, 69] = float("nan"), float("inf")
        r[6, 1] = float("-inf")
        out = gpu_ash.linear(x, w, b, residual=r)
        assert out[3].isnan().all() and not out[5].isfinite().any()
        assert out[6, 1] == float("-inf")
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[3], keep[5], keep[6, 1] = False, False, False
        assert torch.equal(out[keep], plain[keep])
        if dtype != torch.float32:
            assert torch.equal(out[5], torch.where(w[:, 69] > 0, 1.0, -1.0) * float("inf"))


def test_the_same_numbers_every_time(gpu_ash):
    x, w, b, r, gy, u = operands(20_000, 64, 96, torch.float32, seed=9)
    seen = []
    for _ in range(3):
        lx, lw, lb = leaves(x, w, b)
        out = gpu_ash.linear(lx, lw, lb, activation="softplus", scale=100.0, residual=r)
        gx, = torch.autograd.grad(out, lx, gy, create_graph=True)
        got = torch.autograd.grad((out * gy).sum() + (gx * u).sum(), [lx, lw, lb])
        ln, = leaves(torch.linspace(0.5, 1.5, 64, device=DEV))
        gn = torch.autograd.grad(gpu_ash.rms_norm(x, ln), ln, u)
        seen.append([out, gx, *got, *gn])
    for other in seen[1:]:
        assert all(torch.equal(p, q) for p, q in zip(seen[0], other))


def test_rows_beyond_32_bits(gpu_ash):
    """More than 2^31 values in the input and 2^31 bytes of everything else."""
    rows, k, m = (1 << 25) + 5, 64, 33
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(10)
    tail, w = rand(g, 300, k, dtype=torch.bfloat16), rand(g, m, k, size=0.1, dtype=torch.bfloat16)
    x[-300:] = tail
    gy = torch.zeros(rows, m, dtype=torch.bfloat16, device=DEV)
    up = rand(g, 300, m, dtype=torch.bfloat16)
    gy[-300:] = up
    lx, lw = leaves(x, w)
    out = gpu_ash.linear(lx, lw, activation="silu")
    y, d, _, _ = ref.linear(tail, w, None, "silu")
    ref.check(out[-300:], y, torch.bfloat16)
    assert not out[:-300].any()
    gx, gw = torch.autograd.grad(out, [lx, lw], gy)
    want = ref.linear_gradients(up, tail, w, d, "silu", torch.bfloat16)
    ref.check(gx[-300:], want[0], torch.bfloat16)
    ref.check(gw, want[1], torch.bfloat16)
    assert not gx[:-300].any()
    del out, gx, lx, gy
    q = gpu_ash.rms_norm(x, quantize=True)
    assert not q.data[:-300].view(torch.uint8).any() and (q.scales[:-300] == 1).all()
    small = gpu_ash.rms_norm(tail, quantize=True)
    assert torch.equal(q.data[-300:].view(torch.uint8), small.data.view(torch.uint8))
    assert torch.equal(q.scales[-300:], small.scales)


def test_wide_rows_beyond_32_bits(gpu_ash):
    """More than 2^31 values in every operand of the large tiles."""
    rows, k, m, few = 525_000, 4104, 4112, 90
    g = torch.Generator().manual_seed(30)
    at = torch.cat([torch.arange(few // 2), torch.arange(rows - few // 2, rows)]).to(DEV)
    part, up, w = (rand(g, few, k, dtype=torch.bfloat16), rand(g, few, m, dtype=torch.bfloat16),
                   rand(g, m, k, size=k**-0.5, dtype=torch.bfloat16))
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device=DEV)
    x[at] = part
    gy = torch.zeros(rows, m, dtype=torch.bfloat16, device=DEV)
    gy[at] = up
    lx, lw = leaves(x, w)
    out = gpu_ash.linear(lx, lw, activation="silu")
    y, d, _, _ = ref.linear(part, w, None, "silu")
    ref.check(out[at], y, torch.bfloat16)
    assert int(out.any(1).sum()) == few
    gx, gw = torch.autograd.grad(out, [lx, lw], gy)
    want = ref.linear_gradients(up, part, w, d, "silu", torch.bfloat16)
    ref.check(gx[at], want[0], torch.bfloat16)
    ref.check(gw, want[1], torch.bfloat16)
    assert int(gx.any(1).sum()) == few


def test_rows_beyond_one_grid(gpu_ash):
    """More workgroups than a grid holds threads for."""
    rows = (1 << 30) + 77
    x = torch.full((rows, 1), 3.0, dtype=torch.bfloat16, device=DEV)
    x[-5:] = -2.0
    out = gpu_ash.rms_norm(x, eps=7.0)
    assert bool((out[:-5] == 0.75).all()) and bool((out[-5:] == torch.tensor(-2 / 11**0.5).bfloat16().to(DEV)).all())
    lx, = leaves(x)
    gx, = torch.autograd.grad(gpu_ash.rms_norm(lx, eps=7.0), lx, torch.ones_like(x))
    assert bool((gx[:-5] == torch.tensor(7 / 64).bfloat16().to(DEV)).all())
    assert bool((gx[-5:] == torch.tensor(7 / 11**1.5).bfloat16().to(DEV)).all())


def test_the_largest_layer(gpu_ash):
    """65536 features in and out: a weight of 2^32 values."""
    n, rows = 65536, 3
    g = torch.Generator().manual_seed(31)
    w = torch.zeros(n, n, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 1, 777, n // 2 - 1, n // 2, n - 2, n - 1], device=DEV)
    w[at] = rand(g, len(at), n, size=n**-0.5, dtype=torch.bfloat16)
    x, gy = rand(g, rows, n, dtype=torch.bfloat16), rand(g, rows, n, dtype=torch.bfloat16)
    lx, lw = leaves(x, w)
    out = gpu_ash.linear(lx, lw)
    y, d, _, _ = ref.linear(x, w[at], None)
    ref.check(out[:, at], y, torch.bfloat16)
    gx, gw = torch.autograd.grad(out, [lx, lw], gy)
    want = ref.linear_gradients(gy[:, at], x, w[at], d, "none", torch.bfloat16)
    ref.check(gx, want[0], torch.bfloat16)
    ref.check(gw[at], want[1], torch.bfloat16)
    assert bool((gw.view(-1, 8, n)[:, 5, :9] == (gy.double().t() @ x.double()[:, :9]).bfloat16().view(-1, 8, 9)[:, 5]).all())


@pytest.mark.parametrize("rows", [3, 20, 40, 700, 30000])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_what_is_not_finite_in_the_first_row_stays_there(gpu_ash, rows, dtype):
    """Rows and columns beyond the last ones of a tile may be made of the first."""
    x, w, b, _, gy, _ = operands(rows, 70, 40, dtype, seed=32)
    lx, lw, lb = leaves(x, w, b)
    plain = gpu_ash.linear(lx, lw, lb, activation="gelu")
    gx = torch.autograd.grad(plain, lx, gy)[0]
    x, w, b, gy = x.clone(), w.clone(), b.clone(), gy.clone()
    x[0, 0], w[0, 1], b[0], gy[0, 2] = float("nan"), float("nan"), float("inf"), float("nan")
    lx, = leaves(x)
    out = gpu_ash.linear(lx, w, b, activation="gelu")
    assert out[0].isnan().all() and out[:, 0].isnan().all()
    assert torch.equal(out[1:, 1:], plain[1:, 1:])
    w[0, 1] = 0.5   # a finite weight again: the other rows' gradients
    lx, = leaves(x)
    out = gpu_ash.linear(lx, w, None, activation="none")
    clean = torch.autograd.grad(gpu_ash.linear(lx, w, None), lx, torch.nan_to_num(gy))[0]
    got, = torch.autograd.grad(out, lx, gy)
    assert got[0].isnan().all() and torch.equal(got[1:], clean[1:]) and gx.isfinite().all()


# --------------------------------------------------------------------- 8-bit rows
@pytest.mark.parametrize("out_dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1, 16, 1), (1, 1024, 64), (7, 3, 5), (16, 131, 33), (40, 600, 48), (65, 128, 64),
                                   (130, 67, 129), (1000, 257, 300), (16500, 400, 1008), (2500, 272, 1000),
                                   (9000, 2064, 136), (9000, 300, 20), (4000, 131, 200), (17000, 67, 33), (300, 40, 5000)], ids=str)
def test_linear_of_8_bit_rows(gpu_ash, shape, out_dtype):
    rows, k, m = shape
    x, w, b, r, _, _ = operands(rows, k, m, torch.float32, seed=11)
    qx, qw = gpu_ash.QuantizedRows.of(x), gpu_ash.QuantizedRows.of(w)
    b, r = b.to(out_dtype), r.to(out_dtype)
    units8 = out_dtype != torch.float32
    y, _, _, _ = ref.linear(qx.data.float(), qw.data.float(), b, "gelu", 1.0, r, qx.scales, qw.scales, units8)
    ref.check(gpu_ash.linear(qx, qw, b, activation="gelu", residual=r), y, out_dtype)
    y, _, _, _ = ref.linear(qx.data.float(), qw.data.float(), None, "none", 1.0, None, qx.scales, qw.scales, units8)
    ref.check(gpu_ash.linear(qx, qw, out_dtype=out_dtype), y, out_dtype)
    # whole numbers of few bits, whose sums every unit holds: nothing is off but the
    # rounding to the output's type
    g = torch.Generator().manual_seed(18)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g).float().to(DEV)
    wx, ww = whole(rows, k), whole(m, k)
    scales = [torch.randint(0, 3, (n,), generator=g).float().exp2().to(DEV) for n in (rows, m)]
    out = gpu_ash.linear(gpu_ash.QuantizedRows(wx.to(torch.float8_e4m3fn), scales[0]),
                         gpu_ash.QuantizedRows(ww.to(torch.float8_e4m3fn), scales[1]), out_dtype=out_dtype)
    assert torch.equal(out, (wx @ ww.t() * scales[0][:, None] * scales[1]).to(out_dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("width", [1, 7, 64, 513, 2500])
def test_quantized_rows(gpu_ash, width, dtype):
    g = torch.Generator().manual_seed(12)
    x = rand(g, 50, width, dtype=dtype)
    x[3] = 0.0
    x[4] *= 1e-4
    q = gpu_ash.QuantizedRows.of(x)
    most = x.double().abs().amax(1)
    scale = torch.where(most > 0, most / 448.0, 1.0)
    assert q.data.dtype == torch.float8_e4m3fn and q.scales.dtype == torch.float32
    assert ((q.scales.double() - scale).abs() <= 4 * ref.F32 * scale).all()
    v = x.double() / q.scales.double()[:, None]
    # half a step of three bits, or of the numbers below 2^-6; 4 units of float32 beside
    bound = torch.maximum(v.abs() * 2.0**-4, torch.full_like(v, 2.0**-10)) * (1 + 8 * ref.F32)
    assert ((q.data.double() - v).abs() <= bound).all()
    assert (q.dequantize(dtype).double() - x.double()).abs().max() <= most.max() * 2.0**-4 * 1.01
    x[5, width // 2], x[6, 0] = float("nan"), float("inf")
    again = gpu_ash.QuantizedRows.of(x)
    assert again.scales[5].isnan() and again.scales[6].isnan()
    assert again.dequantize()[5:7].isnan().all()
    keep = [i for i in range(50) if i not in (5, 6)]
    assert torch.equal(again.data[keep].view(torch.uint8), q.data[keep].view(torch.uint8))
    assert torch.equal(again.scales[keep], q.scales[keep])


# --------------------------------------------------------------------------- norm
WIDTHS = [1, 3, 8, 31, 33, 64, 67, 130, 256, 300, 512, 777, 1024, 1500, 2048, 2050, 4096, 5000, 8192, 16384]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("width", WIDTHS)
def test_rms_norm_and_its_gradients(gpu_ash, width, dtype):
    g = torch.Generator().manual_seed(13)
    rows, eps = 131 if width < 3000 else 9, 1e-5
    x, r, gy, gs = (rand(g, rows, width, dtype=dtype) for _ in range(4))
    w = (1 + rand(g, width, size=0.2)).to(dtype)
    x[1], r[1] = 0.0, 0.0      # a row of zeros: y = 0, finite gradients
    for residual in (None, r):
        y, i, s = ref.norm(x, w, residual, eps, dtype)
        lx, lw = leaves(x, w)
        lr = None if residual is None else residual.detach().requires_grad_()
        out = gpu_ash.rms_norm(lx, lw, residual=lr, eps=eps)
        if residual is None:
            ref.check(out, y, dtype, "y")
            got = torch.autograd.grad(out, [lx, lw], gy)
            kept = x
        else:
            out, total = out
            ref.check(out, y, dtype, "y")
            ref.check(total, s, dtype, "sum")
            got = torch.autograd.grad([out, total], [lx, lw, lr], [gy, gs])
            assert torch.equal(got[0], got[2])
            kept = total
        # the gradients are those at the sum as it was rounded, which is what is kept
        s = ref.Off(kept)
        _, i = ref.unit(s, eps, w)
        t = ref.Off(gy) * ref.Off(w.expand_as(gy))
        along = (t.v * s.v).mean(1, keepdim=True)
        off = (t.e * s.v.abs()).mean(1, keepdim=True) + (width + 16) * ref.F32 * (t.v * s.v).abs().mean(1, keepdim=True)
        along = ref.Off(along.expand_as(s.v).contiguous(), off.expand_as(s.v).contiguous())
        second = s * (i * (i * (i * along)))
        gx = t * i + ref.Off(-second.v, second.e)
        # the two terms cancel: each is rounded by itself
        gx = ref.Off(gx.v, gx.e + 4 * ref.F32 * ((t * i).v.abs() + second.v.abs()))
        if residual is not None:
            gx = gx + ref.Off(gs)
        ref.check(got[0], gx, dtype, "gx")
        ref.check(got[1], (ref.Off(gy) * (s * i)).column_sums(), dtype, "gw")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("width", [3, 64, 300, 1024, 3000])
@pytest.mark.parametrize("asked", ["x", "xw", "w"])
def test_second_order_of_the_norm(gpu_ash, width, dtype, asked):
    """Against torch's own second order of the plain form in 64 bits.  Its terms are
    sums of up to `width` products (2^-24 each) of unit size with a few roundings to
    the type on the way in and out: 16 half steps of the type, (width + 64) of
    float32, of the gradient's largest row or column."""
    g = torch.Generator().manual_seed(14)
    x, gy, u = (rand(g, 77, width, dtype=dtype) for _ in range(3))
    w, v = (1 + rand(g, width, size=0.2)).to(dtype), rand(g, width, dtype=dtype)

    def second(f, x, w, gy, u, v):
        x, w, gy = leaves(x, w, gy)
        of, ups = {"x": x, "w": w}, {"x": u, "w": v}
        firsts = torch.autograd.grad(f(x, w), [of[n] for n in asked], gy, create_graph=True)
        return torch.autograd.grad(firsts, [gy, x, w], [ups[n] for n in asked], allow_unused=True)

    plain = lambda x, w: x / (x.square().mean(1, keepdim=True) + 1e-6).sqrt() * w
    got = second(lambda x, w: gpu_ash.rms_norm(x, w), x, w, gy, u, v)
    want = second(plain, x.double(), w.double(), gy.double(), u.double(), v.double())
    for have, one, what in zip(got, want, ("gy", "x", "w")):
        if one is None:
            assert have is None or not have.any(), what
            continue
        bound = (16 * ref.half(dtype) + (width + 64) * ref.F32) * one.abs()
        size = one.norm(dim=-1, keepdim=True) if one.dim() == 2 else one.norm()
        assert have.dtype == dtype
        assert ((have.double() - one).abs() <= bound + (16 * ref.half(dtype) + (width + 64) * ref.F32) * size).all(), what


def test_norm_layouts(gpu_ash):
    g = torch.Generator().manual_seed(15)
    wide, w = rand(g, 40, 100), rand(g, 67)
    for x in (wide[:, 3:70], rand(g, 67, 40).t(), wide[:1, :67].expand(40, 67), wide[5, 1:68], rand(g, 2, 4, 67)):
        r = rand(g, 67)
        flat = x.reshape(-1, 67)
        y, _, s = ref.norm(flat, w, r.expand_as(flat), 1e-6, torch.float32)
        lx, lr = leaves(x, r)
        out, total = gpu_ash.rms_norm(lx, w, residual=lr)
        assert out.shape == total.shape == x.shape
        ref.check(out.reshape(-1, 67), y, torch.float32)
        ref.check(total.reshape(-1, 67), s, torch.float32)
        gx, gr = torch.autograd.grad(out.sum(), [lx, lr])
        assert torch.allclose(gx.reshape(-1, 67).sum(0), gr, rtol=1e-4, atol=1e-4)
        # only the sum is used
        _, total = gpu_ash.rms_norm(lx, w, residual=lr)
        gx, = torch.autograd.grad(total.sum(), lx)
        assert (gx == 1).all()


def test_norm_in_8_bits_is_the_norm_rounded(gpu_ash):
    g = torch.Generator().manual_seed(16)
    for rows, width, dtype in ((1, 1024, torch.bfloat16), (100, 67, torch.float32), (50, 3000, torch.float16)):
        x, r, w = rand(g, rows, width, dtype=dtype), rand(g, rows, width, dtype=dtype), rand(g, width, dtype=dtype)
        q, total = gpu_ash.rms_norm(x, w, residual=r, quantize=True)
        _, want = gpu_ash.rms_norm(x, w, residual=r)
        assert torch.equal(total, want)
        y, _, _ = ref.norm(x, w, r, 1e-6, dtype)
        scale = y.v.abs().amax(1) / 448
        off = y.e.amax(1) / 448 + 4 * ref.F32 * scale
        assert ((q.scales.double() - scale).abs() <= off).all()
        v = y.v / q.scales.double()[:, None]
        bound = torch.maximum(v.abs() * 2.0**-4, torch.full_like(v, 2.0**-10)) + 2 * y.e / q.scales.double()[:, None]
        assert ((q.data.double() - v).abs() <= bound * 1.0001).all()


# -------------------------------------------------------------------- as they are used
def decoder_loss(decoder, grid, x):
    x = x.detach().requires_grad_()
    features, _ = grid(x, "smooth_step")
    y = decoder(torch.cat([features, x], 1))
    gx, = torch.autograd.grad(y[:, 0].sum(), x, create_graph=True)
    return y.square().mean() + 0.1 * (gx.norm(dim=1) - 1).abs().mean(), y


class PlainDecoder:
    """A FeatureDecoder's weights through torch's operations."""

    def __init__(self, decoder):
        self.d = decoder

    def __call__(self, rows):
        d, f = self.d, torch.nn.functional
        act = {"softplus": lambda z: f.softplus(d.scale * z, threshold=1e9) / d.scale, "sine": lambda z: torch.sin(d.scale * z)}[d.activation]
        norm = lambda h, w: h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt() * w
        layer = lambda one, h: f.linear(h, one["weight"], one["bias"])
        h = act(layer(d.first, rows))
        for i, (up, down) in enumerate(zip(d.up, d.down)):
            h = h + layer(down, act(layer(up, norm(h, d.norms[i]))))
        return layer(d.last, norm(h, d.norms[-1]))


@pytest.mark.parametrize("activation,scale,blocks", [("softplus", 10.0, 2), ("sine", 3.0, 1), ("softplus", 1.0, 0)])
def test_decoder_on_a_grid_with_an_eikonal_loss(gpu_ash, activation, scale, blocks):
    import workloads

    torch.manual_seed(0)
    grid, radii, centres = workloads.build_grid(gpu_ash, 300, 8, sparse_grid_dim=32, device=DEV)
    x = workloads.ray_queries(grid, radii, centres, num_rays=20, samples_per_ray=33)
    decoder = gpu_ash.FeatureDecoder(11, 4, width=48, blocks=blocks, activation=activation, scale=scale, device=DEV)
    params = [grid.embeddings, *decoder.parameters()]
    loss, y = decoder_loss(decoder, grid, x)
    got = torch.autograd.grad(loss, params)
    want_loss, want_y = decoder_loss(PlainDecoder(decoder), grid, x)
    want = torch.autograd.grad(want_loss, params)
    # float32 on both sides, a dozen layers' worth of roundings of 2^-24 a term and up
    # to 660 terms a sum
    assert torch.allclose(y, want_y, rtol=1e-4, atol=1e-4 * float(want_y.abs().max()))
    assert abs(float(loss - want_loss)) <= 1e-4 * abs(float(want_loss))
    for p, q in zip(got, want):
        assert float((p - q).norm()) <= 1e-3 * float(q.norm()) + 1e-9


def test_decoder_in_8_bits(gpu_ash):
    torch.manual_seed(1)
    decoder = gpu_ash.FeatureDecoder(19, 4, width=128, blocks=2, activation="silu", device=DEV)
    x = torch.randn(500, 19, device=DEV)
    with torch.no_grad():
        want = decoder(x)
        got = decoder.quantize_()(x)
        assert torch.equal(decoder.dequantize_()(x), want)
    # two roundings of 2^-4 of a term (row and weight) in each of four products, which
    # add up as the root of their number
    assert float((got - want).norm()) <= 4 * 2 * 2.0**-4 * float(want.norm())
    with pytest.raises(RuntimeError, match="no gradients"):
        decoder.quantize_()(x)


def test_on_another_stream_and_in_a_graph(gpu_ash):
    """A training step (features, eikonal-like second order) and a served step,
    captured and replayed on new inputs between eager work."""
    g = torch.Generator().manual_seed(17)
    x, w, b, n = rand(g, 700, 67), rand(g, 64, 67, size=0.1), rand(g, 64), 1 + rand(g, 64, size=0.1)
    gy, u = rand(g, 700, 64), rand(g, 700, 67)
    lx, lw, lb, ln = leaves(x, w, b, n)
    q8 = gpu_ash.QuantizedRows.of(rand(g, 32, 64))

    def step():
        y = gpu_ash.linear(lx, lw, lb, activation="softplus", scale=10.0)
        y, total = gpu_ash.rms_norm(y, ln, residual=y)
        gx, = torch.autograd.grad(y, lx, gy, create_graph=True)
        grads = torch.autograd.grad([gx, y], [lx, lw, lb, ln], [u, gy])
        with torch.no_grad():
            served = gpu_ash.linear(gpu_ash.rms_norm(total.detach(), ln, quantize=True), q8, out_dtype=torch.float32)
        return [y, gx, *grads, served]

    eager = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(eager, on_side))
    del on_side
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        g = torch.Generator().manual_seed(100 + seed)
        with torch.no_grad():
            lx.copy_(rand(g, 700, 67))
        eager = [t.detach().clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, captured)), seed


def test_a_capture_beside_an_eager_graph_of_the_same_leaves_is_refused(gpu_ash):
    """Only the forward is captured here: that is where it is refused."""
    x, w = leaves(torch.randn(40, 8, device=DEV), torch.randn(8, 8, device=DEV))
    n = torch.ones(8, device=DEV, requires_grad=True)
    kept = gpu_ash.rms_norm(gpu_ash.linear(x, w), n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for call in (lambda: gpu_ash.linear(x, w), lambda: gpu_ash.rms_norm(x.detach(), n)):
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            with pytest.raises(RuntimeError, match="still holds these leaves"):
                call()
            graph.capture_end()
    torch.cuda.synchronize()
    del kept
    out = gpu_ash.linear(x, w)
    assert torch.autograd.grad(out.sum(), x)[0].shape == x.shape


def test_a_broadcast_residual_with_a_gradient_is_not_captured(gpu_ash):
    x, w, r = torch.randn(40, 8, device=DEV), torch.randn(8, 8, device=DEV), torch.randn(8, device=DEV)
    lr, = leaves(r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for call in (lambda: gpu_ash.linear(x, w, residual=lr), lambda: gpu_ash.rms_norm(x, residual=lr)):
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            graph.capture_begin()
            with pytest.raises(RuntimeError, match="broadcast residual"):
                call()
            kept = gpu_ash.linear(x, w, residual=r)
            graph.capture_end()
        torch.cuda.synchronize()
        del kept
    assert torch.autograd.grad(gpu_ash.linear(x, w, residual=lr).sum(), lr)[0].tolist() == [40.0] * 8


def test_third_order_is_refused(gpu_ash):
    x, w, u = leaves(torch.randn(5, 4, device=DEV), torch.randn(3, 4, device=DEV), torch.randn(5, 4, device=DEV))
    gx, = torch.autograd.grad(gpu_ash.linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="third order"):
        torch.autograd.grad(gx, w, u, create_graph=True)
    gx, = torch.autograd.grad(gpu_ash.rms_norm(x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="third order"):
        torch.autograd.grad(gx, x, u, create_graph=True)
