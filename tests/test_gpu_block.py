"""GPU: the gated residual step with its norms (edgehip.block) against its formula in fp64 under automatic
differentiation, and against differences.

Tolerances.  An output is rounded once: half a step, eps/2 of the value.  What is rounded is fp32 arithmetic, whose error
`bounds` carries through the formulas row by row from the sizes of the terms: each stage (a subtraction, product or sum)
adds at most K 2^-24 of its terms' size, K = 24 (its own few roundings, and a row's sum: at most 8 values a thread, 10
levels of pairs), to what its operands are off by, scaled as they are scaled.  A sum over rows adds the rows' errors and
at most 128 roundings of partial sums (rows per thread <= 64, 64 partials)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)]


def step(t):
    return torch.finfo(t).eps / 2 if t != F32 else 0.0


def make(rows, dim, types=(F32, F32), kind='rms', gate='none', groups=4, seed=0, pre=True, post=True, behind=0, ptype=F32, gtype=None):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def n(*s):
        return torch.randn(*s, generator=g, device='cuda')
    th, tz = types
    v = dict(h=(2 * n(rows, dim)).to(th), z=(n(rows, dim) + 0.3).to(tz))
    opts = dict(kind=kind, pre=pre, post=post, res_scale=0.75, eps=1e-5)
    if pre:
        v['w_pre'] = (1 + 0.2 * n(dim)).to(ptype)
    if post:
        v['w_post'] = (1 + 0.2 * n(dim)).to(ptype)
    if kind == 'layer':
        if pre:
            v['b_pre'] = (0.2 * n(dim)).to(ptype)
        if post:
            v['b_post'] = (0.2 * n(dim)).to(ptype)
    row_ptr = None
    if gate == 'vector':
        v['gate'] = n(dim).to(gtype or F32)
    elif gate == 'row':
        v['gate'] = n(rows, dim).to(gtype or tz)
    elif gate == 'group':
        v['gate'] = n(groups, dim).to(gtype or F32)
        cut = torch.randint(0, rows - behind + 1, (groups - 1,), generator=g, device='cuda').sort().values
        row_ptr = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), rows - behind)]).to(torch.int32)
    return v, row_ptr, opts


def formula(v, row_ptr, opts):
    def norm(x, w, b):
        if opts['kind'] == 'layer':
            x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + opts['eps'])
        x = x * w
        return x if b is None else x + b
    u = norm(v['z'], v['w_post'], v.get('b_post')) if opts['post'] else v['z']
    g = v.get('gate', 1.0)
    if row_ptr is not None:
        own = torch.repeat_interleave(torch.arange(len(row_ptr) - 1, device=u.device), (row_ptr[1:] - row_ptr[:-1]).long())
        spread = g[own]
        g = torch.cat([spread, spread.new_zeros(u.shape[0] - len(own), u.shape[1])])
    h = opts['res_scale'] * v['h'] + g * u
    return h, norm(h, v['w_pre'], v.get('b_pre')) if opts['pre'] else None


def reference(v, row_ptr, opts, dh, dy):
    d = {k: t.detach().double().requires_grad_(True) for k, t in v.items()}
    h, y = formula(d, row_ptr, opts)
    out = [(h, dh)] + ([(y, dy)] if y is not None and dy is not None else [])
    out = [(o, g) for o, g in out if g is not None]
    grads = torch.autograd.grad([o for o, _ in out], list(d.values()), [g.double() for _, g in out], allow_unused=True)
    return h.detach(), None if y is None else y.detach(), dict(zip(d, grads))


K = 24 * U


def bounds(v, row_ptr, opts, dh, dy):
    """How far each output and gradient may be from the formula: per row [rows, 1], per column sums [1] or [groups, 1]."""
    d = {k: t.double() for k, t in v.items()}
    rows = d['h'].shape[0]
    top = lambda x: x.abs().amax(-1, keepdim=True)
    one = torch.ones(rows, 1, dtype=torch.float64, device='cuda')

    def stats(x):
        mean = x.mean(-1, keepdim=True) if opts['kind'] == 'layer' else 0.0
        r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + opts['eps'])
        return r, top((x - mean) * r), top(x) + (mean.abs() if opts['kind'] == 'layer' else 0.0)
    wz, wh = (float(d[k].abs().max()) if k in d else 1.0 for k in ('w_post', 'w_pre'))
    bz, bh = (float(d[k].abs().max()) if k in d else 0.0 for k in ('b_post', 'b_pre'))
    g = float(d['gate'].abs().max()) if 'gate' in d else 1.0
    rz, zh, tz = stats(d['z'])
    ez = K * (2 * tz * rz * (1 + zh) + zh)                       # zhat: the difference, and 1 / size (off by tz rz relative)
    u, eu = (zh * wz + bz, ez * wz + K * (zh * wz + bz)) if opts['post'] else (top(d['z']), 0 * one)
    th = opts['res_scale'] * top(d['h']) + g * u
    eh = g * eu + K * th
    h64, _ = formula(d, row_ptr, opts)
    rh, hh, mh = stats(h64)
    rel = rh * (eh + K * mh)                                     # of 1 / size
    ehh = 2 * rel * (1 + hh) + K * hh
    out = dict(h=eh, y=ehh * wh + K * (hh * wh + bh))
    ty = top(dy.double()) if dy is not None else 0 * one
    nt = rh * ty * wh * (2 + hh) if opts['pre'] else 0 * one
    en = nt * (K + rel) + rh * ty * wh * ehh * (1 + hh) if opts['pre'] else 0 * one
    D = (top(dh.double()) if dh is not None else 0 * one) + nt
    eD = en + K * D
    s, es = D * g, eD * g + K * D * g
    if opts['post']:
        relz = K + K * tz * rz
        dz = rz * wz * (es * (2 + zh) + s * ez * (1 + zh) + s * (2 + zh) * relz)
    else:
        dz = es
    sums = lambda e, size: (e + 128 * U * size).sum(0)
    out.update(dh=opts['res_scale'] * eD + K * D, dz=dz, dw_pre=sums(ty * ehh, ty * hh), db_pre=sums(K * ty, ty),
               dw_post=sums(es * zh + s * ez, s * zh), db_post=sums(es, s))
    eg = eD * u + D * eu + K * D * u
    if row_ptr is not None:
        own = torch.repeat_interleave(torch.arange(len(row_ptr) - 1, device='cuda'), (row_ptr[1:] - row_ptr[:-1]).long())
        out['dgate'] = torch.zeros(len(row_ptr) - 1, 1, dtype=torch.float64, device='cuda').index_add_(0, own, (eg + 128 * U * D * u)[:len(own)])
    elif 'gate' in d:
        out['dgate'] = sums(eg, D * u) if d['gate'].dim() == 1 else eg
    return out


def near(got, want, tol, what):
    assert got.shape == want.shape, what
    if want.numel() == 0:
        return
    tol = step(got.dtype) * (want.abs() + tol) + tol + (2.0 ** -25 if got.dtype == F16 else 1e-40)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


def check(v, row_ptr, opts, dh, dy):
    """The differentiable form: outputs and every gradient."""
    import edgehip
    leaves = {k: t.detach().clone().requires_grad_(True) for k, t in v.items()}
    h, y = edgehip.gate_norm(leaves['h'], leaves['z'], row_ptr=row_ptr, **{k: t for k, t in leaves.items() if k not in 'hz'}, **opts)
    outs = [(h, dh)] + ([(y, dy)] if y is not None else [])
    outs = [(o, g) for o, g in outs if g is not None]
    grads = dict(zip(leaves, torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)))
    rh, ry, rg = reference(v, row_ptr, opts, dh, dy)
    assert h.dtype == v['h'].dtype and (y is None) == (not opts['pre'])
    if v['h'].shape[0] == 0:
        for k, g in grads.items():
            assert g.shape == v[k].shape and not bool(g.any()), k
        return h, y, grads
    tol = bounds(v, row_ptr, opts, dh, dy)
    near(h, rh, tol['h'], 'h')
    if y is not None:
        assert y.dtype == v['z'].dtype
        near(y, ry, tol['y'], 'y')
    for k, want in rg.items():
        got = grads[k]
        if want is None:
            assert got is None or not bool(got.any()), k
            continue
        assert got.dtype == v[k].dtype and got.shape == v[k].shape, k
        near(got, want, tol['d' + k], 'd' + k)
    return h, y, grads


def gradients(v, opts, seed=1, dtype_scale=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    dh = (torch.randn(v['h'].shape, generator=g, device='cuda') * dtype_scale).to(v['h'].dtype)
    dy = (torch.randn(v['z'].shape, generator=g, device='cuda') * dtype_scale).to(v['z'].dtype) if opts['pre'] else None
    return dh, dy


@pytest.mark.parametrize('dim', [1, 2, 7, 8, 9, 63, 64, 65, 100, 128, 129, 257, 513, 1023, 1024, 1101, 2049, 4096, 5000, 8192])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
def test_widths(dim, kind):
    for rows, gate in ((1, 'vector'), (37, 'group')):
        v, ptr, opts = make(rows, dim, kind=kind, gate=gate, seed=dim)
        check(v, ptr, opts, *gradients(v, opts))


@pytest.mark.parametrize('types', TYPES)
@pytest.mark.parametrize('gate', ['none', 'vector', 'group', 'row'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
def test_types_and_gates(types, gate, kind):
    for dim in (64, 333, 1536):
        v, ptr, opts = make(70, dim, types=types, kind=kind, gate=gate, seed=dim)
        check(v, ptr, opts, *gradients(v, opts))
        v, ptr, opts = make(70, dim, types=types, kind=kind, gate=gate, seed=dim, ptype=types[1], gtype=types[1])
        check(v, ptr, opts, *gradients(v, opts))


@pytest.mark.parametrize('gate', ['none', 'vector', 'group', 'row'])
@pytest.mark.parametrize('pre,post', [(True, False), (False, True), (False, False)])
def test_a_norm_switched_off(gate, pre, post):
    v, ptr, opts = make(50, 200, kind='layer', gate=gate, pre=pre, post=post)
    check(v, ptr, opts, *gradients(v, opts))


def test_many_rows_and_groups():
    for rows, dim, groups in ((5000, 64, 300), (4097, 24, 4097), (3000, 520, 2), (2500, 64, 1)):
        v, ptr, opts = make(rows, dim, kind='layer', gate='group', groups=groups, seed=rows)
        check(v, ptr, opts, *gradients(v, opts))
    v, ptr, opts = make(20000, 40, gate='vector')
    check(v, ptr, opts, *gradients(v, opts))


def test_rows_behind_the_last_group_pass_as_the_residual():
    v, ptr, opts = make(100, 96, gate='group', groups=5, behind=30)
    h, _, grads = check(v, ptr, opts, *gradients(v, opts))
    assert torch.equal(h[70:], 0.75 * v['h'][70:])
    assert not bool(grads['z'][70:].any())


def test_only_one_output_used():
    v, ptr, opts = make(33, 72, kind='layer', gate='group')
    dh, dy = gradients(v, opts)
    check(v, ptr, opts, dh, None)
    check(v, ptr, opts, None, dy)


def test_no_rows():
    v, ptr, opts = make(0, 32, kind='layer', gate='group', groups=3)
    h, y, _ = check(v, ptr, opts, *gradients(v, opts))
    assert h.shape == (0, 32) and y.shape == (0, 32)


def test_higher_dimensions_strides_and_offsets():
    import edgehip
    v, _, opts = make(60, 100, types=(BF16, BF16), gate='row')
    wide_h, wide_z = torch.randn(60, 211, device='cuda').to(BF16), torch.randn(60, 207, device='cuda').to(BF16)
    h, z = wide_h[:, 11:111], wide_z[:, 3:103]                   # rows that start at odd addresses
    ref = edgehip.gate_norm(h.clone(), z.clone(), w_pre=v['w_pre'], w_post=v['w_post'], gate=v['gate'], **opts)
    got = edgehip.gate_norm(h, z, w_pre=v['w_pre'], w_post=v['w_post'], gate=v['gate'], **opts)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    got = edgehip.gate_norm(h.reshape(3, 20, 100), z.reshape(3, 20, 100), w_pre=v['w_pre'], w_post=v['w_post'],
                            gate=v['gate'].view(3, 20, 100), **opts)
    assert torch.equal(got[0].view(60, 100), ref[0]) and torch.equal(got[1].view(60, 100), ref[1])
    # dense tensors at an address no vector is aligned to
    base = torch.randn(60 * 100 + 1, device='cuda').to(BF16)
    off = base[1:].view(60, 100)
    assert off.data_ptr() % 16
    got = edgehip.gate_norm(off, z, w_pre=v['w_pre'], w_post=v['w_post'], gate=v['gate'], **opts)
    ref = edgehip.gate_norm(off.clone(), z.clone(), w_pre=v['w_pre'], w_post=v['w_post'], gate=v['gate'], **opts)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_values_far_from_one():
    """A row of zeros, a constant row, rows near the ends of the range; an infinity or NaN stays in its row."""
    v, ptr, opts = make(12, 128, kind='layer', gate='vector')
    v['z'][0], v['z'][1], v['h'][1] = 0.0, 3.0, 0.0
    v['z'][2] *= 1e-12
    v['h'][3] *= 1e15
    import edgehip
    kw = {k: t for k, t in v.items() if k not in 'hz'}
    h, y = edgehip.gate_norm(v['h'], v['z'], **kw, **opts)
    rh, ry = formula({k: t.double() for k, t in v.items()}, ptr, opts)
    scale = rh.abs().amax(1, keepdim=True) + 4
    assert bool(((h.double() - rh).abs() <= 64 * U * scale).all())
    assert bool(((y.double() - ry).abs() <= 256 * U * (ry.abs().amax(1, keepdim=True) + 8)).all())
    v['z'][5, 7], v['h'][6, 1] = float('inf'), float('nan')
    h2, y2 = edgehip.gate_norm(v['h'], v['z'], **kw, **opts)
    ok = [i for i in range(12) if i not in (5, 6)]
    assert torch.equal(h2[ok], h[ok]) and torch.equal(y2[ok], y[ok])
    assert bool(y2[5].isnan().all()) and bool(y2[6].isnan().all())


@pytest.mark.parametrize('gate', ['vector', 'group', 'row'])
def test_against_differences(gate):
    """Directional differences in fp32: step 2^-5; the formula's third derivatives are O(1) per value, so the difference
    is off by ~2^-10 of the direction's size, the rounding of the outputs adds 2^-24 x 2^5 each: 1 % of the product."""
    import edgehip
    v, ptr, opts = make(40, 48, kind='layer', gate=gate)
    dh, dy = gradients(v, opts)
    _, _, grads = check(v, ptr, opts, dh, dy)
    gen = torch.Generator(device='cuda').manual_seed(5)
    for k in v:
        d = torch.randn(v[k].shape, generator=gen, device='cuda')
        e = 2.0 ** -5 / float(d.norm()) * v[k].shape[-1] ** 0.5
        val = []
        for sign in (1, -1):
            w = dict(v)
            w[k] = v[k] + sign * e * d
            h, y = edgehip.gate_norm(w['h'], w['z'], row_ptr=ptr, **{a: b for a, b in w.items() if a not in 'hz'}, **opts)
            val.append(float((h.double() * dh.double()).sum() + (y.double() * dy.double()).sum()))
        diff, want = (val[0] - val[1]) / (2 * e), float((grads[k].double() * d.double()).sum())
        size = float(grads[k].double().norm() * d.double().norm())
        assert abs(diff - want) <= 0.01 * size, (k, diff, want, size)


def test_same_bits_each_time_on_other_streams_and_in_a_graph():
    import edgehip.block as block
    v, ptr, opts = make(700, 192, types=(F32, BF16), kind='layer', gate='group', groups=9)
    dh, dy = gradients(v, opts)
    kw = {k: t for k, t in v.items() if k not in 'hz'}

    def both():
        h, y, stats = block.gate_norm_fwd(v['h'], v['z'], row_ptr=ptr, want_stats=True, **kw, **opts)
        return [h, y] + list(block.gate_norm_bwd(dh, dy, v['h'], v['z'], stats, row_ptr=ptr, **kw, **opts).values())
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
        v['z'].copy_(torch.randn(v['z'].shape, device='cuda') + k)
        graph.replay()
        torch.cuda.synchronize()
        want = both()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k
