"""GPU: 8-bit activation checkpoints (edgehip.ckpt8): codes and exponents against their definition exactly, the passes
that read them against fp64 on the kept values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def step(t):
    return torch.finfo(t).eps / 2 if t != F32 else 0.0


def kept64(x):
    """The definition: the smallest e of [-120, 121] with max|x| <= 127 2^e (else 121), whole multiples to nearest even
    within +-127."""
    m, k = x.shape
    kg = -(-k // 64)
    v = torch.zeros(m, kg * 64, dtype=torch.float64)
    v[:, :k] = x.double().cpu()
    v = v.view(m, kg, 64)
    steps = torch.tensor([2.0 ** i for i in range(-120, 122)], dtype=torch.float64)
    bad = ~torch.isfinite(v).all(2)
    top = torch.where(bad, 0.0, v.abs().amax(2))
    e = torch.searchsorted(127 * steps, top.contiguous()).clamp(max=241)
    s = steps[e][:, :, None]
    codes = torch.where(bad[:, :, None], 0.0, torch.round(v / s).clamp(-127, 127))
    value = torch.where(bad[:, :, None], torch.nan, codes * s).view(m, -1)[:, :k]
    return codes.view(m, -1)[:, :k], torch.where(bad, -128, e - 120), value


def sample(m, k, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(m, k, generator=g, device='cuda') * torch.exp(2 * torch.randn(m, 1, generator=g, device='cuda'))
    if m > 3:
        x[1] = 0
        x[2] *= 1e-6 if dtype == F16 else 1e-30
    return x.to(dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('k', [1, 5, 8, 63, 64, 65, 127, 128, 130, 200, 1000, 1024])
def test_codes_and_exponents_are_the_definition(dtype, k):
    import edgehip
    for m in (1, 33, 300):
        x = sample(m, k, dtype, seed=k)
        p = edgehip.pack8(x)
        codes, exps, value = kept64(x)
        assert p.codes.shape == x.shape and p.exps.shape == (m, -(-k // 64))
        assert torch.equal(p.codes.cpu().double(), codes) and torch.equal(p.exps.cpu().long(), exps)
        assert torch.equal(p.unpack(F32).cpu().double(), value)
        # bf16 holds every kept value
        assert torch.equal(p.unpack(BF16).cpu().double(), value)
        assert p.unpack().dtype == dtype


def test_borders_of_the_exponent_ties_and_extremes():
    import edgehip
    rows = []
    for top in (127.0, 127.00001, 126.99999, 128.0, 1.0, 0.9921875, 0.99218756, 3.4028234663852886e38, 1e-38, 1e-45, 2.0 ** -113):
        r = torch.zeros(64, dtype=F32)
        r[0], r[1], r[2], r[3] = top, -top / 2, top / 254, 0.5
        if top < 1e-30 or top > 1e30:
            r[3] = 0
        rows.append(r)
    r = torch.arange(-32, 32, dtype=F32) + 0.5                    # ties, with 127 as the largest: step 1
    r[0] = 127
    rows.append(r)
    x = torch.stack(rows).cuda()
    p = edgehip.pack8(x)
    codes, exps, value = kept64(x)
    assert torch.equal(p.exps.cpu().long(), exps)
    assert torch.equal(p.codes.cpu().double(), codes)
    assert torch.equal(p.unpack().cpu().double(), value)
    assert bool(((value - x.cpu().double()).abs() <= x.cpu().double().abs().amax(1, keepdim=True) / 127 + 2.0 ** -121).all())


def test_what_is_not_finite_stays_visible():
    import edgehip
    x = sample(6, 200, F32)
    x[2, 70], x[3, 199], x[4, 0] = float('nan'), float('inf'), float('-inf')
    p = edgehip.pack8(x)
    v = p.unpack().cpu()
    bad = torch.zeros(6, 200, dtype=torch.bool)
    bad[2, 64:128] = bad[3, 192:] = bad[4, :64] = True
    assert torch.equal(v.isnan(), bad)
    dw, db = edgehip.ckpt8.linear8_bwd_weight(torch.ones(6, 3, device='cuda'), p)
    assert torch.equal(dw.cpu().isnan(), bad.any(0).expand(3, 200)) and bool(torch.isfinite(db).all())
    dx = edgehip.ckpt8.act8_bwd(torch.ones_like(x), p)
    assert torch.equal(dx.cpu().isnan(), bad)


def act64(kind):
    return torch.nn.functional.silu if kind == 'silu' else torch.nn.functional.mish


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('kind', ['silu', 'mish'])
def test_activations(dtype, kind):
    """y: half a step and ~10 fp32 operations on terms of |x|; dx: the derivative is at most 1.1 and made of terms of
    1 + |x|, ~16 operations."""
    import edgehip
    for m, k in ((1, 1), (40, 100), (33, 64), (200, 384)):
        x = (sample(m, k, dtype, seed=k) * 2).clamp(-60, 60)
        y, p = edgehip.ckpt8.act8_fwd(x, kind)
        want = act64(kind)(x.double())
        assert y.dtype == dtype
        assert bool(((y.double() - want).abs() <= step(dtype) * want.abs() + 16 * U * x.double().abs() + 2.0 ** -126 + (2.0 ** -25 if dtype == F16 else 0)).all())
        assert torch.equal(p.codes, edgehip.pack8(x).codes) and torch.equal(p.exps, edgehip.pack8(x).exps)
        dy = torch.randn(m, k, device='cuda').to(dtype)
        q = p.unpack(F32).double().requires_grad_(True)
        (want,) = torch.autograd.grad(act64(kind)(q), q, dy.double())
        for got in (edgehip.ckpt8.act8_bwd(dy, p, kind),
                    torch.autograd.grad(edgehip.act8(leaf := x.clone().requires_grad_(True), kind), leaf, dy)[0]):
            assert got.dtype == dtype
            tol = step(dtype) * want.abs() + 32 * U * dy.double().abs() * (1 + q.detach().abs()) + (2.0 ** -25 if dtype == F16 else 0)
            assert bool(((got.double() - want).abs() <= tol).all())


def test_activation_far_from_zero():
    import edgehip
    x = torch.tensor([[-1e30, -200.0, -88.0, -20.0, 20.0, 88.0, 200.0, 1e30, 0.0, -0.0]], device='cuda')
    for kind in ('silu', 'mish'):
        y, p = edgehip.ckpt8.act8_fwd(x, kind)
        want = act64(kind)(x.double())
        assert bool(((y.double() - want).abs() <= 16 * U * x.double().abs().clamp(max=100) * (x.double() < 0) + 16 * U * want.abs() + 1e-35).all()), (kind, y)
        dx = edgehip.ckpt8.act8_bwd(torch.ones_like(x), p, kind)
        assert bool(torch.isfinite(dx).all()) and float(dx[0, 7]) == 1.0 and float(dx[0, 0]) == 0.0


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n,k', [(1, 1, 1), (1, 64, 64), (31, 5, 3), (32, 128, 128), (33, 129, 65), (777, 99, 130), (500, 192, 64),
                                   (2048, 256, 64), (3001, 70, 333), (4100, 130, 257), (9000, 64, 64)])
def test_weight_gradient(dtype, m, n, k):
    """Products are exact; a sum of m terms in fp32 is off by at most its number of additions, here bounded by m / 16 + 64
    (matrix instructions add 16 rows at a time, splits and partials follow), times 2^-24 of the sum of the sizes.  (The
    additions inside one instruction are counted as roundings too: 16 + m / 16.)"""
    import edgehip
    x, dy = sample(m, k, dtype, seed=m), torch.randn(m, n, device='cuda').to(dtype)
    p = edgehip.pack8(x)
    dw, db = edgehip.ckpt8.linear8_bwd_weight(dy, p)
    q = p.unpack(F32).double().cpu()
    d = dy.double().cpu()
    want, size = d.t() @ q, d.abs().t() @ q.abs()
    ops = m / 16 + 80
    assert dw.dtype == F32 and bool(((dw.double().cpu() - want).abs() <= ops * U * size + 1e-30).all())
    assert bool(((db.double().cpu() - d.sum(0)).abs() <= (m / 8 + 80) * U * d.abs().sum(0)).all())
    again, db2 = edgehip.ckpt8.linear8_bwd_weight(dy, p)
    assert torch.equal(again, dw) and torch.equal(db, db2)
    only, none = edgehip.ckpt8.linear8_bwd_weight(dy, p, bias=False)
    assert none is None and torch.equal(only, dw)


@pytest.mark.parametrize('dtype', TYPES)
def test_weight_gradient_sees_infinities_and_tiny_gradients(dtype):
    import edgehip
    x = torch.randn(70, 64, device='cuda').to(dtype)
    dy = torch.randn(70, 40, device='cuda').to(dtype)
    dy[:, 3] = 2.0 ** -24 if dtype == F16 else 2.0 ** -120
    dy[9, 5], dy[8, 6] = float('inf'), float('nan')
    p = edgehip.pack8(x)
    dw, db = edgehip.ckpt8.linear8_bwd_weight(dy, p)
    q = p.unpack(F32).double()
    fine = [i for i in range(40) if i not in (5, 6)]
    want = dy.double().t()[fine] @ q
    size = dy.double().abs().t()[fine] @ q.abs()
    assert bool(((dw[fine].double() - want).abs() <= 90 * U * size).all())
    assert not bool(torch.isfinite(dw[5]).any()) and bool(dw[6].isnan().all())
    assert float(db[5]) == float('inf') and bool(db[6].isnan())


def test_no_rows_give_zero_gradients():
    import edgehip
    p = edgehip.pack8(torch.zeros(0, 70, device='cuda'))
    dw, db = edgehip.ckpt8.linear8_bwd_weight(torch.zeros(0, 9, device='cuda'), p)
    assert dw.shape == (9, 70) and not bool(dw.any()) and not bool(db.any())
    assert p.unpack().shape == (0, 70)
    x = torch.zeros(0, 70, device='cuda', requires_grad=True)
    edgehip.act8(x).sum().backward()
    assert x.grad.shape == (0, 70)


@pytest.mark.parametrize('dtype,n,k', [(F32, 64, 128), (F32, 30, 50), (BF16, 64, 128), (F16, 24, 72)])
def test_linear_layer(dtype, n, k):
    """Forward and input gradient are those of the exact input; the weight's gradient those of the kept one."""
    import edgehip
    x = torch.randn(5, 30, k, device='cuda').to(dtype) if dtype != F32 else torch.randn(150, k, device='cuda')
    w, b = (torch.randn(n, k, device='cuda') * k ** -0.5).to(dtype), torch.randn(n, device='cuda').to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = edgehip.linear8(*leaves)
    dy = torch.randn_like(y)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x2, dy2 = x.reshape(-1, k).double(), dy.reshape(-1, n).double()
    tol = lambda want, size, ops: step(dtype) * want.abs() + ops * U * size + (2.0 ** -25 if dtype == F16 else 0)
    want = x2 @ w.double().t() + b.double()
    assert bool(((y.reshape(-1, n).double() - want).abs() <= tol(want, x2.abs() @ w.double().abs().t() + b.double().abs(), k + 8)).all())
    want = dy2 @ w.double()
    assert bool(((dx.reshape(-1, k).double() - want).abs() <= tol(want, dy2.abs() @ w.double().abs(), n + 8)).all())
    q = edgehip.pack8(x).unpack(F32).reshape(-1, k).double()
    want = dy2.t().contiguous() @ q
    assert dw.dtype == dtype and bool(((dw.double() - want).abs() <= tol(want, dy2.abs().t().contiguous() @ q.abs(), 100)).all())
    want = dy2.sum(0)
    assert bool(((db.double() - want).abs() <= tol(want, dy2.abs().sum(0), 100)).all())
    # a shared checkpoint, a layer whose weight is fixed, and no gradient at all
    kept = edgehip.pack8(x)
    y2 = edgehip.linear8(leaves[0], leaves[1], leaves[2], kept)
    assert torch.equal(torch.autograd.grad(y2, leaves[1], dy)[0], dw)
    y3 = edgehip.linear8(leaves[0], w, leaves[2])
    dx3, db3 = torch.autograd.grad(y3, [leaves[0], leaves[2]], dy)
    assert torch.equal(dx3, dx) and bool(((db3.double() - db.double()).abs() <= 2 * tol(db.double(), dy2.abs().sum(0), 100)).all())
    with torch.no_grad():
        assert torch.equal(edgehip.linear8(*leaves), y)


def test_gradients_against_differences():
    """The activation's and the layer's gradients through kept values are those of a loss of the kept values: a directional
    difference of that loss (fp64), step 2^-12: third derivatives O(1), fp32 gradients to 1e-6."""
    import edgehip
    x, dy = sample(30, 96, F32).clamp(-8, 8), torch.randn(30, 96, device='cuda')
    p = edgehip.pack8(x)
    q, d = p.unpack().double(), torch.randn(30, 96, device='cuda').double()
    e = 2.0 ** -12
    for kind in ('silu', 'mish'):
        got = float((edgehip.ckpt8.act8_bwd(dy, p, kind).double() * d).sum())
        f = [float((act64(kind)(q + s * e * d) * dy.double()).sum()) for s in (1, -1)]
        size = float(dy.double().norm() * d.norm())
        assert abs((f[0] - f[1]) / (2 * e) - got) <= 1e-5 * size


def test_other_streams_and_graphs():
    import edgehip
    x, dy = torch.randn(3000, 160, device='cuda').to(BF16), torch.randn(3000, 96, device='cuda').to(BF16)

    def both():
        y, p = edgehip.ckpt8.act8_fwd(x)
        return [y, p.codes, p.exps, edgehip.ckpt8.act8_bwd(y, p)] + list(edgehip.ckpt8.linear8_bwd_weight(dy, p))
    ref = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(3):
        x.copy_(torch.randn(x.shape, device='cuda') * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both())), k


def test_an_infinity_in_the_last_row_and_one_long_row():
    import edgehip
    x = torch.rand(45, 64, device='cuda').to(BF16) + 0.5
    dy = torch.ones(45, 40, device='cuda').to(BF16)
    dy[44, 7] = float('inf')
    dw, db = edgehip.ckpt8.linear8_bwd_weight(dy, edgehip.pack8(x))
    assert bool((dw[7] == float('inf')).all()) and float(db[7]) == float('inf')
    assert bool(torch.isfinite(dw[torch.arange(40) != 7]).all())
    long = sample(1, (1 << 20) + 37, F32, seed=9)[0]
    p = edgehip.pack8(long)
    codes, exps, value = kept64(long[None])
    assert p.shape == long.shape and torch.equal(p.exps.cpu().long(), exps) and torch.equal(p.unpack().cpu().double(), value[0])


def test_a_layer_whose_weight_is_fixed_captured():
    """Only the bias learns: its gradient, replayed with eager work between, is the eager one each time."""
    import edgehip
    x, dy = torch.randn(40000, 96, device='cuda').to(BF16), torch.randn(40000, 200, device='cuda').to(BF16)
    w, b = torch.randn(200, 96, device='cuda').to(BF16), torch.zeros(200, device='cuda').to(BF16)

    def run():
        leaf = b.detach().requires_grad_(True)
        return torch.autograd.grad(edgehip.linear8(x, w, leaf), leaf, dy)[0]
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(4):
        dy.copy_(torch.randn(dy.shape, device='cuda') * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run()), k
        want = dy.double().sum(0)
        # fp32 sums in two levels of a few hundred terms each, one rounding to bf16
        assert bool(((out.double() - want).abs() <= step(BF16) * want.abs() + 1000 * U * dy.double().abs().sum(0)).all()), k


@pytest.mark.parametrize('shift', [0, 1, 2, 3])
def test_a_layer_on_views_that_start_anywhere(shift):
    import edgehip
    m, n, k = 70, 64, 128

    def view(r, c, seed):
        flat = torch.randn(r * c + 4, generator=torch.Generator(device='cuda').manual_seed(seed), device='cuda')
        return flat[shift:shift + r * c].view(r, c)
    x, w, dy, b = view(m, k, 1), view(n, k, 2), view(m, n, 3), view(1, n, 4)[0]
    got, want = [], []
    for out, form in ((got, lambda t: t), (want, lambda t: t.clone())):
        leaves = [form(t).detach().requires_grad_(True) for t in (x, w, b)]
        y = edgehip.linear8(*leaves)
        out += [y.detach()] + list(torch.autograd.grad(y, leaves, form(dy)))
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_a_layer_keeps_its_type_inside_autocast():
    import edgehip
    x = torch.randn(33, 50, device='cuda').requires_grad_(True)
    w = torch.randn(30, 50, device='cuda').requires_grad_(True)
    y = edgehip.linear8(x, w)
    with torch.autocast('cuda', dtype=BF16):
        z = edgehip.linear8(x, w)
        grads = torch.autograd.grad(z, [x, w], torch.ones_like(z))
    assert z.dtype == F32 and torch.equal(y, z)
    assert all(torch.equal(a, c) for a, c in zip(grads, torch.autograd.grad(y, [x, w], torch.ones_like(y))))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('m,n,k', [(1030, 4099, 4100), (70001, 300, 500), (66000, 1000, 257), (131101, 129, 258), (70000, 512, 256), (9001, 300, 500),
                                   (129, 700, 1100), (300, 2048, 513)])
def test_weight_gradient_large(dtype, m, n, k):
    """Products large enough for the larger tile, and some just below; tolerances as above."""
    import edgehip
    x, dy = sample(m, k, dtype, seed=m), torch.randn(m, n, device='cuda').to(dtype)
    p = edgehip.pack8(x)
    dw, db = edgehip.ckpt8.linear8_bwd_weight(dy, p)
    q, d = p.unpack(F32).double(), dy.double()
    want, size = d.t().contiguous() @ q, d.abs().t().contiguous() @ q.abs()
    assert bool(((dw.double() - want).abs() <= (m / 16 + 80) * U * size + 1e-30).all())
    assert bool(((db.double() - d.sum(0)).abs() <= (m / 8 + 80) * U * d.abs().sum(0)).all())
    again, db2 = edgehip.ckpt8.linear8_bwd_weight(dy, p)
    assert torch.equal(again, dw) and torch.equal(db, db2)
